// Rules on rows of logits before a draw: penalties for tokens that the text holds, biases of single tokens, a mask of
// allowed ones (bmb_logits_adjust).
//
// One pass over the logits.  A block has a part of a row's vocabulary; what the text holds of that part is counted in shared memory
// first, from the whole text (from L2: it is short beside the row).  Bound by memory where rows are many; so a block's logits are
// on their way to its registers before it counts, and 3 or 4 blocks an SM have enough of them in flight.  Counts are whole numbers and
// of biases the last entry holds, so no order of the atomics shows.
#include "common.cuh"
#include <climits>

namespace bmb {
namespace {

constexpr int LG_THREADS = 512, LG_EACH = 8, LG_PART = LG_THREADS * LG_EACH;

__global__ void __launch_bounds__(LG_THREADS, 3) adjust_k(float *out, const float *logits, int V, long long stride, int parts, const __grid_constant__ bmb_logit_rules r) {
    // per token of this block's part: how often it was drawn, with SEEN where the text holds it; and the last bias entry for it, from 1
    __shared__ int count[LG_PART], last[LG_PART];
    constexpr int SEEN = 1 << 31;
    const int row = blockIdx.x / parts, v0 = (blockIdx.x % parts) * LG_PART, size = min(LG_PART, V - v0);
    if (r.history)
#pragma unroll
        for (int k = 0; k < LG_EACH / 4; ++k) reinterpret_cast<int4 *>(count)[threadIdx.x + k * LG_THREADS] = make_int4(0, 0, 0, 0);
    if (r.bias_ids)
#pragma unroll
        for (int k = 0; k < LG_EACH / 4; ++k) reinterpret_cast<int4 *>(last)[threadIdx.x + k * LG_THREADS] = make_int4(0, 0, 0, 0);
    let_successor_start();
    wait_for_predecessor();
    float x[LG_EACH];
    unsigned words[LG_EACH];
    const float *from = logits + (size_t)row * stride + v0;
#pragma unroll
    for (int k = 0; k < LG_EACH; ++k) {
        const int i = threadIdx.x + k * LG_THREADS;
        x[k] = i < size ? from[i] : 0.0f;
        words[k] = i < size && r.allowed ? r.allowed[(size_t)row * r.allowed_stride + ((v0 + i) >> 5)] : ~0u;
    }
    const float rep = r.repetition ? r.repetition[row] : 1.0f, freq = r.frequency ? r.frequency[row] : 0.0f, pres = r.presence ? r.presence[row] : 0.0f;
    __syncthreads();
    constexpr int AHEAD = 4;
    if (r.history) {
        const int len = min(max(r.history_lens[row], 0), r.history_stride), prompt = r.prompt_lens ? r.prompt_lens[row] : 0;
        const int *text = r.history + (size_t)row * r.history_stride;
        for (int j0 = threadIdx.x; j0 < len; j0 += AHEAD * LG_THREADS) {
            int token[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) token[k] = j0 + k * LG_THREADS < len ? text[j0 + k * LG_THREADS] : -1;
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int at = token[k] - v0;                 // (a token below 0 is below v0)
                if (token[k] < 0 || at < 0 || at >= size) continue;
                if (j0 + k * LG_THREADS >= prompt) atomicAdd(&count[at], 1);
                atomicOr(&count[at], SEEN);
            }
        }
    }
    if (r.bias_ids) {
        const int len = min(max(r.bias_lens[row], 0), r.bias_stride);
        const int *ids = r.bias_ids + (size_t)row * r.bias_stride;
        for (int j = threadIdx.x; j < len; j += LG_THREADS) {
            const int id = ids[j], at = id - v0;
            if (id >= 0 && at >= 0 && at < size) atomicMax(&last[at], j + 1);
        }
    }
    __syncthreads();
    float *to = out + (size_t)row * stride + v0;
#pragma unroll
    for (int k = 0; k < LG_EACH; ++k) {
        const int i = threadIdx.x + k * LG_THREADS;
        if (i >= size) break;
        const int c = r.history ? count[i] : 0, b = r.bias_ids ? last[i] : 0;
        if (c) {
            const int drawn = c & ~SEEN;
            if (r.repetition) x[k] = x[k] > 0.0f ? __fdiv_rn(x[k], rep) : __fmul_rn(x[k], rep);
            if (drawn) x[k] = __fsub_rn(__fsub_rn(x[k], __fmul_rn(freq, (float)drawn)), pres);
        }
        if (b) x[k] = __fadd_rn(x[k], r.bias[(size_t)row * r.bias_stride + b - 1]);
        if (!(words[k] >> ((v0 + i) & 31) & 1)) x[k] = -INFINITY;
        to[i] = x[k];
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
    return launch_in_chain(adjust_k, n * parts, LG_THREADS, 0, (cudaStream_t)stream, out, logits, V, stride, parts, r);
}
