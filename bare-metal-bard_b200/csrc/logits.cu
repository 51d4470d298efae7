// Rules on rows of logits before a draw: penalties for tokens that the text holds, biases of single tokens, a mask of
// allowed ones (bmb_logits_adjust).
//
// One pass over the logits, a part of a row's vocabulary a block.  The part and the mask's words come to shared memory by cp.async while what the
// text holds of the part is counted there (from the whole text, which is in L2: it is short beside the row); each token found for the first time goes
// on a list, of which one thread each works out the new value in place, then biases are added, and the pass that stores the part, 4 elements at a
// time, has only the mask left to do.  Bound by memory where rows are many, if nothing that a rule needs comes from farther than shared memory and an
// element that no rule touches costs few instructions.  256 rows of 50257, us: 16.8 with next to no text (15.7 being what the memory takes), 18.9 with texts of
// up to 1024 tokens, 21.8 with 64 biases and a mask too, 5 blocks an SM, the issue slots two thirds in use; with the part read from L2 once its text was counted 17.1, 20.8 and
// 28.4, 8 and 5 blocks an SM; with no list, each token's new value worked out by a thread that finds it in a second walk over the text, 16.9, 18.4 and
// 22.2, but texts beyond 1024 tokens are then read twice (20 thousand tokens: 98 with the list).  Counts are whole numbers, of biases the last entry holds, and the list's order does
// not matter, so no order of the atomics shows.
#include "common.cuh"
#include <climits>
#include <type_traits>

namespace bmb {
namespace {

constexpr int LG_THREADS = 256, LG_FOURS = 4, LG_PART = LG_THREADS * LG_FOURS * 4, LG_BLOCKS = 5;

__device__ __forceinline__ void copy16(void *to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(void *to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// VEC: logits and out have the same offset from a 16-byte boundary, so that a row's elements can be taken 4 at a time from its first
// boundary on: parts begin `shift` elements before multiples of LG_PART.
template <bool VEC>
__global__ void __launch_bounds__(LG_THREADS, LG_BLOCKS) adjust_k(float *out, const float *logits, int V, long long stride, int parts, const __grid_constant__ bmb_logit_rules r) {
    // the part; of each of its tokens 2 for each time it was drawn and 1 if it is in the prompt, and later its last bias entry, from 1; the
    // tokens of the text in a list; the mask's words
    __shared__ __align__(16) float part[LG_PART];
    extern __shared__ __align__(16) unsigned count[];
    unsigned short *list = reinterpret_cast<unsigned short *>(count + LG_PART);
    __shared__ unsigned mask[LG_PART / 32 + 2];
    __shared__ int listed;
    static_assert(LG_PART <= 1 << 16, "");
    const bool ruled = r.history || r.bias_ids;
    if (ruled)
#pragma unroll
        for (int k = 0; k < LG_FOURS; ++k) reinterpret_cast<uint4 *>(count)[threadIdx.x + k * LG_THREADS] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    let_successor_start();
    wait_for_predecessor();
    const int row = blockIdx.x / parts;
    const float *from = logits + row * stride;
    const int v0 = (blockIdx.x - row * parts) * LG_PART - (VEC ? (int)((uintptr_t)from >> 2 & 3) : 0);      // (at most 3 before the row's first)
    const bool inner = v0 >= 0 && v0 + LG_PART <= V;
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
    if (r.bias_ids) {
        if ((int)threadIdx.x < r.bias_stride) {
            id = ids[threadIdx.x];
            bias = r.bias[(size_t)row * r.bias_stride + threadIdx.x];
        }
        biases = r.bias_lens[row];
    }
    // each(place in the part, elements: 4, or 1 where they are not side by side on a boundary in memory, or partly outside the row)
    auto elements = [&](auto &&each) {
#pragma unroll
        for (int k = 0; k < LG_FOURS * (VEC ? 1 : 4); ++k) {
            const int i = (threadIdx.x + k * LG_THREADS) * (VEC ? 4 : 1), v = v0 + i;
            if (VEC && (inner || (v >= 0 && v + 3 < V))) {
                each(i, std::integral_constant<int, 4>());
            } else {
#pragma unroll
                for (int e = 0; e < (VEC ? 4 : 1); ++e)
                    if (v + e >= 0 && v + e < V) each(i + e, std::integral_constant<int, 1>());
            }
        }
    };
    elements([&](int i, auto n) {
        if constexpr (decltype(n)::value == 4) copy16(part + i, from + v0 + i);
        else copy4(part + i, from + v0 + i);
    });
    // (from the word that has the part's first element on; of the first part, words before the row's first do not matter)
    const int w0 = v0 >> 5;
    if (r.allowed)
        for (int i = threadIdx.x; i < LG_PART / 32 + 2; i += LG_THREADS)
            if (w0 + i >= 0 && 32 * (w0 + i) < V) copy4(mask + i, r.allowed + (size_t)row * r.allowed_stride + w0 + i);
    // the part's tokens: `span` of them from `least` on
    const int least = max(v0, 0);
    const unsigned span = max(min(v0 + LG_PART, V) - least, 0);      // (the last part may begin behind the row)
    len = min(max(len, 0), r.history_stride);
    biases = min(max(biases, 0), r.bias_stride);
    for (int j = 4 * threadIdx.x; j < len; j += 4 * LG_THREADS) {
        const int t[4] = {token.x, token.y, token.z, token.w};
        read_text(j + 4 * LG_THREADS, len);                   // (ahead of these ones' counting)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if ((unsigned)t[e] - (unsigned)least >= span || j + e >= len) continue;
            const int at = t[e] - v0;
            const unsigned before = j + e >= prompt ? atomicAdd(&count[at], 2u) : atomicOr(&count[at], 1u);
            if (before == 0) list[atomicAdd(&listed, 1)] = (unsigned short)at;
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    for (int i = threadIdx.x; i < listed; i += LG_THREADS) {
        const int at = list[i], drawn = (int)(count[at] >> 1);
        float y = part[at];
        if (r.repetition) y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
        if (drawn && r.frequency) y = __fsub_rn(y, __fmul_rn(freq, (float)drawn));
        if (drawn && r.presence) y = __fsub_rn(y, pres);
        part[at] = y;
        count[at] = 0;
    }
    if (r.bias_ids) {
        // use(place in the part, index) of each bias that the part has
        auto entries = [&](auto &&use) {
            for (int j = threadIdx.x; j < biases; j += LG_THREADS) {
                const int v = j < LG_THREADS ? id : ids[j];
                if ((unsigned)v - (unsigned)least < span) use(v - v0, j);
            }
        };
        __syncthreads();
        entries([&](int at, int j) { atomicMax(&count[at], j + 1u); });
        __syncthreads();
        entries([&](int at, int j) {
            if (count[at] == j + 1u) part[at] = __fadd_rn(part[at], j < LG_THREADS ? bias : r.bias[(size_t)row * r.bias_stride + j]);
        });
    }
    __syncthreads();
    float *to = out + row * stride + v0;
    elements([&](int i, auto n) {
        constexpr int N = decltype(n)::value;
        float x[N];
        if constexpr (N == 4) *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(part + i);
        else x[0] = part[i];
        if (r.allowed) {
            const int v = v0 + i, w = (v >> 5) - w0;
            const unsigned allowed = __funnelshift_r(mask[w], mask[w + 1], v & 31);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (!(allowed >> e & 1)) x[e] = -INFINITY;
        }
        if constexpr (N == 4) *reinterpret_cast<float4 *>(to + i) = *reinterpret_cast<const float4 *>(x);
        else to[i] = x[0];
    });
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
    const size_t smem = r.history || r.bias_ids ? LG_PART * 6 : 0;
    static_assert(LG_PART * 10 + 1024 <= 48 * 1024, "");      // (more would have to be asked for)
    auto kernel = vec ? adjust_k<true> : adjust_k<false>;
    return launch_in_chain(kernel, n * parts, LG_THREADS, smem, (cudaStream_t)stream, out, logits, V, stride, parts, r);
}
