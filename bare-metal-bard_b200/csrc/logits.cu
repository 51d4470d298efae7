// Rules on rows of logits before a draw: penalties for tokens that the text holds, biases of single tokens, a mask of
// allowed ones (bmb_logits_adjust).
//
// One pass over the logits; what a text holds is counted in shared memory first, a block's part of the vocabulary at a time.
#include "common.cuh"
#include <climits>

namespace bmb {
namespace {

constexpr int LG_THREADS = 512, LG_PART = 4096;

__global__ void __launch_bounds__(LG_THREADS) adjust_k(float *out, const float *logits, int V, long long stride, int parts, bmb_logit_rules r) {
    // per token of this block's part: how often it was drawn, with SEEN where the text holds it; and the last bias entry for it, from 1
    __shared__ int count[LG_PART], last[LG_PART];
    constexpr int SEEN = 1 << 31;
    const int row = blockIdx.x / parts, v0 = (blockIdx.x % parts) * LG_PART, size = min(LG_PART, V - v0);
    for (int i = threadIdx.x; i < size; i += LG_THREADS) count[i] = last[i] = 0;
    __syncthreads();
    if (r.history) {
        const int len = min(max(r.history_lens[row], 0), r.history_stride), prompt = r.prompt_lens ? r.prompt_lens[row] : 0;
        const int *text = r.history + (size_t)row * r.history_stride;
        for (int j = threadIdx.x; j < len; j += LG_THREADS) {
            const unsigned at = (unsigned)text[j] - (unsigned)v0;
            if (text[j] < 0 || at >= (unsigned)size) continue;
            atomicOr(&count[at], SEEN);
            if (j >= prompt) atomicAdd(&count[at], 1);
        }
    }
    if (r.bias_ids) {
        const int len = min(max(r.bias_lens[row], 0), r.bias_stride);
        const int *ids = r.bias_ids + (size_t)row * r.bias_stride;
        for (int j = threadIdx.x; j < len; j += LG_THREADS) {
            const unsigned at = (unsigned)ids[j] - (unsigned)v0;
            if (ids[j] >= 0 && at < (unsigned)size) atomicMax(&last[at], j + 1);
        }
    }
    __syncthreads();
    const float rep = r.repetition ? r.repetition[row] : 1.0f, freq = r.frequency ? r.frequency[row] : 0.0f, pres = r.presence ? r.presence[row] : 0.0f;
    for (int i = threadIdx.x; i < size; i += LG_THREADS) {
        const int v = v0 + i;
        float x = logits[(size_t)row * stride + v];
        const int c = count[i];
        if (c) {
            const int drawn = c & ~SEEN;
            if (r.repetition) x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
            if (drawn) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)drawn)), pres);
        }
        if (last[i]) x = __fadd_rn(x, r.bias[(size_t)row * r.bias_stride + last[i] - 1]);
        if (r.allowed && !(r.allowed[(size_t)row * r.allowed_stride + (v >> 5)] >> (v & 31) & 1)) x = -INFINITY;
        out[(size_t)row * stride + v] = x;
    }
}

}  // namespace
}  // namespace bmb

using namespace bmb;

extern "C" int bmb_logits_adjust(float *out, const float *logits, int n, int V, long long stride, const bmb_logit_rules *rules, void *stream) {
    if (!rules || n < 0 || V < 0 || stride < V) return fail(BMB_E_ARG, "logits_adjust: bad argument (n=%d V=%d stride=%lld)", n, V, stride);
    if (n == 0 || V == 0) return BMB_OK;
    const bmb_logit_rules &r = *rules;
    if (!out || !logits) return fail(BMB_E_ARG, "logits_adjust: a null pointer");
    if (!r.history && (r.repetition || r.frequency || r.presence)) return fail(BMB_E_ARG, "logits_adjust: penalties need a history");
    if (r.history && (!r.history_lens || r.history_stride < 0)) return fail(BMB_E_ARG, "logits_adjust: a history needs history_lens and a stride");
    if (!r.bias_ids != !r.bias || (r.bias_ids && (!r.bias_lens || r.bias_stride < 0)))
        return fail(BMB_E_ARG, "logits_adjust: biases need bias_ids, bias, bias_lens and a stride");
    if (r.allowed && r.allowed_stride < (V + 31LL) / 32) return fail(BMB_E_ARG, "logits_adjust: %d words are no mask of %d tokens", r.allowed_stride, V);
    const int parts = ceil_div(V, LG_PART);
    if ((long long)n * parts > INT_MAX) return fail(BMB_E_LIMIT, "logits_adjust: %d rows of %d", n, V);
    return launch(false, adjust_k, n * parts, LG_THREADS, 0, (cudaStream_t)stream, out, logits, V, stride, parts, r);
}
