// Rules on rows of logits before a draw: penalties for tokens that the text holds, biases of single tokens, a mask of
// allowed ones (bmb_logits_adjust).
//
// One pass over the logits, a part of a row's vocabulary a block.  What the text holds of the part is counted in shared memory, from the
// whole text (from L2: it is short beside the row); each token found for the first time goes on a list, of which one thread each works out
// the new value, and the pass over the part, 4 elements at a time, only picks those up.  Bound by memory where rows are many, if an element
// that no rule touches costs few instructions: with the rules' arithmetic in the pass itself some lane of most warps needed
// it, and 256 rows of 50257 took 41 us, the issue slots full.  The logits go to L2 first, while the counting waits for the text: held in registers
// meanwhile they left room for half the blocks.  Counts are whole numbers, of biases the last entry holds, and the list's order does not
// matter, so no order of the atomics shows.  256 rows of 50257, us: 17.1 with next to no text (15.7 being what the memory takes), 20.8 with texts of
// up to 1024 tokens, 28.4 with 64 biases and a mask too: the steps between a block's barriers, which other blocks have to fill.
#include "common.cuh"
#include <climits>

namespace bmb {
namespace {

constexpr int LG_THREADS = 256, LG_FOURS = 4, LG_PART = LG_THREADS * LG_FOURS * 4;

// VEC: logits and out have the same offset from a 16-byte boundary, so that a row's elements can be taken 4 at a time from its first
// boundary on: parts begin `shift` elements before multiples of LG_PART.
// BIASES: shared memory for them, and with it 5 blocks an SM instead of 8.
template <bool VEC, bool BIASES>
__global__ void __launch_bounds__(LG_THREADS, BIASES ? 5 : 8) adjust_k(float *out, const float *logits, int V, long long stride, int parts, const __grid_constant__ bmb_logit_rules r) {
    // of the part, which tokens have a bias and which are in the text, a bit each; the mask's words; how often each token was drawn, and then
    // its new value; those of the text in a list; the last bias entry for each, from 1.
    constexpr int WORDS = LG_PART / 32;
    extern __shared__ __align__(16) unsigned shared[];
    __shared__ unsigned with_bias[WORDS], seen[WORDS], mask[WORDS + 2];
    __shared__ int listed;
    int *count = reinterpret_cast<int *>(shared);
    float *value = reinterpret_cast<float *>(shared);
    unsigned short *list = reinterpret_cast<unsigned short *>(count + LG_PART);
    int *last = reinterpret_cast<int *>(list + LG_PART);      // (only where there are biases)
    bool ruled = r.history || BIASES;
    if (ruled) {
        for (int i = threadIdx.x; i < WORDS; i += LG_THREADS) with_bias[i] = seen[i] = 0;
#pragma unroll
        for (int k = 0; k < LG_FOURS; ++k) {
            reinterpret_cast<int4 *>(count)[threadIdx.x + k * LG_THREADS] = make_int4(0, 0, 0, 0);
            if (BIASES) reinterpret_cast<int4 *>(last)[threadIdx.x + k * LG_THREADS] = make_int4(0, 0, 0, 0);
        }
        if (threadIdx.x == 0) listed = 0;
    }
    static_assert(LG_PART <= 1 << 16, "");
    let_successor_start();
    wait_for_predecessor();
    const int row = blockIdx.x / parts;
    const float *from = logits + row * stride;
    const int v0 = (blockIdx.x - row * parts) * LG_PART - (VEC ? (int)((uintptr_t)from >> 2 & 3) : 0);      // (at most 3 before the row's first)
    const bool inner = VEC && v0 >= 0 && v0 + LG_PART <= V;
    // the part on its way to L2, 128 bytes a thread
    for (int v = v0 + 32 * (int)threadIdx.x; v < min(v0 + LG_PART, V); v += 32 * LG_THREADS)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(from + max(v, 0)));
    const int *text = r.history + (size_t)row * r.history_stride, *ids = r.bias_ids + (size_t)row * r.bias_stride;
    int4 token;
    int id = -1, len = 0, prompt = 0, biases = 0;
    float bias = 0.0f, rep = 1.0f, freq = 0.0f, pres = 0.0f;
    auto read_text = [&](int j, int len) {                    // 4 tokens from j on; -1 from `len` on
        token = make_int4(-1, -1, -1, -1);
        if (j + 3 < len && ((uintptr_t)(text + j) & 15) == 0) {
            token = *reinterpret_cast<const int4 *>(text + j);
        } else {
            if (j < len) token.x = text[j];
            if (j + 1 < len) token.y = text[j + 1];
            if (j + 2 < len) token.z = text[j + 2];
            if (j + 3 < len) token.w = text[j + 3];
        }
    };
    if (r.history) {
        read_text(4 * threadIdx.x, r.history_stride);
        len = r.history_lens[row];
        prompt = r.prompt_lens ? r.prompt_lens[row] : 0;
        if (r.repetition) rep = r.repetition[row];
        if (r.frequency) freq = r.frequency[row];
        if (r.presence) pres = r.presence[row];
    }
    if (BIASES) {
        if ((int)threadIdx.x < r.bias_stride) {
            id = ids[threadIdx.x];
            bias = r.bias[(size_t)row * r.bias_stride + threadIdx.x];
        }
        biases = r.bias_lens[row];
    }
    // (from the word that has the part's first element on; of the first part, words before the row's first do not matter)
    const int w0 = v0 >> 5;
    if (r.allowed)
        for (int i = threadIdx.x; i < WORDS + 2; i += LG_THREADS)
            mask[i] = w0 + i >= 0 && 32 * (w0 + i) < V ? r.allowed[(size_t)row * r.allowed_stride + w0 + i] : 0u;
    __syncthreads();
    // the part's tokens: `span` of them from `least` on
    const int least = max(v0, 0);
    const unsigned span = max(min(v0 + LG_PART, V) - least, 0);      // (the last part may begin behind the row)
    const auto bit = [](int at) { return 1u << (at & 31); };
    // use(place in the part, index) of each bias that the part has
    auto entries = [&](auto &&use) {
        for (int j = threadIdx.x; BIASES && j < biases; j += LG_THREADS) {
            const int v = j < LG_THREADS ? id : ids[j];
            if ((unsigned)v - (unsigned)least < span) use(v - v0, j);
        }
    };
    if (ruled) {
        len = min(max(len, 0), r.history_stride);
        biases = min(max(biases, 0), r.bias_stride);
        bool found = false;
        for (int j = 4 * threadIdx.x; j < len; j += 4 * LG_THREADS) {
            if (j >= 4 * LG_THREADS) read_text(j, len);
            const int t[4] = {token.x, token.y, token.z, token.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if ((unsigned)t[e] - (unsigned)least >= span || j + e >= len) continue;
                const int at = t[e] - v0;
                found = true;
                if (j + e >= prompt) atomicAdd(&count[at], 1);
                if (!(atomicOr(&seen[at >> 5], bit(at)) & bit(at))) list[atomicAdd(&listed, 1)] = (unsigned short)at;
            }
        }
        entries([&](int at, int j) {
            found = true;
            atomicMax(&last[at], j + 1);
            atomicOr(&with_bias[at >> 5], bit(at));
        });
        ruled = __syncthreads_or(found);                      // (nothing: the rest is a copy)
    }
    if (ruled) {
        // those with a bias by the thread of its last entry, the others of the text from the list
        auto penalised = [&](int at) {
            const int drawn = count[at];
            float y = from[v0 + at];
            if (r.repetition) y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
            if (drawn && r.frequency) y = __fsub_rn(y, __fmul_rn(freq, (float)drawn));
            if (drawn && r.presence) y = __fsub_rn(y, pres);
            return y;
        };
        entries([&](int at, int j) {
            if (last[at] != j + 1) return;
            const float y = seen[at >> 5] & bit(at) ? penalised(at) : from[v0 + at];
            value[at] = __fadd_rn(y, j < LG_THREADS ? bias : r.bias[(size_t)row * r.bias_stride + j]);
        });
        // (from the last thread down: the warps that have no bias first)
        for (int i = LG_THREADS - 1 - threadIdx.x; i < listed; i += LG_THREADS)
            if (!(with_bias[list[i] >> 5] & bit(list[i]))) value[list[i]] = penalised(list[i]);
        __syncthreads();
    }
    float *to = out + row * stride;
    float x[LG_FOURS][4];
#pragma unroll
    for (int k = 0; k < LG_FOURS; ++k) {
        const int v = v0 + 4 * (threadIdx.x + k * LG_THREADS);
        if (inner || (VEC && v >= 0 && v + 3 < V)) {
            *reinterpret_cast<float4 *>(x[k]) = *reinterpret_cast<const float4 *>(from + v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[k][e] = v + e >= 0 && v + e < V ? from[v + e] : 0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < LG_FOURS; ++k) {
        const int i = 4 * (threadIdx.x + k * LG_THREADS), v = v0 + i;
        if (ruled) {
            const unsigned marks = (with_bias[i >> 5] | seen[i >> 5]) >> (i & 31) & 15;
            if (marks) {
                const float4 y = *reinterpret_cast<const float4 *>(value + i);
                if (marks & 1) x[k][0] = y.x;
                if (marks & 2) x[k][1] = y.y;
                if (marks & 4) x[k][2] = y.z;
                if (marks & 8) x[k][3] = y.w;
            }
        }
        if (r.allowed) {
            const int w = (v >> 5) - w0;
            const unsigned allowed = __funnelshift_r(mask[w], mask[w + 1], v & 31);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!(allowed >> e & 1)) x[k][e] = -INFINITY;
        }
        if (inner || (VEC && v >= 0 && v + 3 < V)) {
            *reinterpret_cast<float4 *>(to + v) = *reinterpret_cast<const float4 *>(x[k]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v + e >= 0 && v + e < V) to[v + e] = x[k][e];
        }
    }
}

}  // namespace
}  // namespace bmb

using namespace bmb;

extern "C" int bmb_logits_adjust(float *out, const float *logits, int n, int V, long long stride, const bmb_logit_rules *rules, void *stream) {
    if (!rules || n < 0 || V < 0 || stride < V) return fail(BMB_E_ARG, "logits_adjust: bad argument (n=%d V=%d stride=%lld)", n, V, stride);
    if (n == 0 || V == 0) return BMB_OK;
    const bmb_logit_rules &r = *rules;
    if (!out || !logits || !words(out, logits, r.history, r.history_lens, r.prompt_lens, r.repetition, r.frequency, r.presence, r.bias_ids, r.bias, r.bias_lens, r.allowed))
        return fail(BMB_E_ARG, "logits_adjust: a null or unaligned pointer");
    if (!r.history && (r.repetition || r.frequency || r.presence)) return fail(BMB_E_ARG, "logits_adjust: penalties need a history");
    if (r.history && (!r.history_lens || r.history_stride < 0)) return fail(BMB_E_ARG, "logits_adjust: a history needs history_lens and a stride");
    if (!r.bias_ids != !r.bias || (r.bias_ids && (!r.bias_lens || r.bias_stride < 0)))
        return fail(BMB_E_ARG, "logits_adjust: biases need bias_ids, bias, bias_lens and a stride");
    if (r.allowed && r.allowed_stride < (V + 31LL) / 32) return fail(BMB_E_ARG, "logits_adjust: %d words are no mask of %d tokens", r.allowed_stride, V);
    if (r.history_stride > 1 << 30 || r.bias_stride > 1 << 30) return fail(BMB_E_LIMIT, "logits_adjust: rows of more than 2^30 tokens or biases");
    const bool vec = (((uintptr_t)out ^ (uintptr_t)logits) & 15) == 0;
    const int parts = ceil_div(V + (vec ? 3LL : 0LL), LG_PART);
    if ((long long)n * parts > INT_MAX || V > INT_MAX - 2 * LG_PART) return fail(BMB_E_LIMIT, "logits_adjust: %d rows of %d", n, V);
    const size_t smem = (r.history || r.bias_ids ? LG_PART * 6 : 0) + (r.bias_ids ? LG_PART * 4 : 0);
    static_assert(LG_PART * 10 <= 48 * 1024, "");             // (more would have to be asked for)
    auto kernel = r.bias_ids ? vec ? adjust_k<true, true> : adjust_k<false, true> : vec ? adjust_k<true, false> : adjust_k<false, false>;
    return launch_in_chain(kernel, n * parts, LG_THREADS, smem, (cudaStream_t)stream, out, logits, V, stride, parts, r);
}
