// A paged cache of keys and values, and attention of one new token of each request over its pages.
#include "common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <climits>
#include <cmath>

namespace bmb {
namespace {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

template <typename T>
__global__ void __launch_bounds__(256) kv_write_k(bmb_kv_cache c, const float *k, const float *v, long long row_stride, const int *slots) {
    const int slot = slots[blockIdx.x];
    if (slot < 0 || slot >= c.pages * c.page_size) return;
    const long long page = slot / c.page_size, off = slot % c.page_size;
    for (int e = threadIdx.x; e < c.heads * c.head_size; e += blockDim.x) {
        const long long from = blockIdx.x * row_stride + e;
        const long long to = page * c.page_stride + off * c.token_stride + (e / c.head_size) * c.head_stride + e % c.head_size;
        ((T *)c.k)[to] = from_float<T>(k[from]);
        ((T *)c.v)[to] = from_float<T>(v[from]);
    }
}

// A block for each request and query head; its warps take tokens in turn, a lane HS / 32 elements of each.
template <typename T, int HS>
__global__ void __launch_bounds__(256) attend_k(float *out, float *lse, const float *q, bmb_kv_cache c, const int *tables, const int *lens, int heads,
                                                long long q_stride, long long out_stride, int max_pages, float scale) {
    constexpr int E = HS / 32, WARPS = 8;
    __shared__ float m_of[WARPS], l_of[WARPS], o_of[WARPS][HS];
    const int i = blockIdx.x / heads, h = blockIdx.x % heads, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int len = (int)min((long long)max(lens[i], 0), (long long)max_pages * c.page_size);
    const T *K = (const T *)c.k + (h / (heads / c.heads)) * c.head_stride, *V = (const T *)c.v + (h / (heads / c.heads)) * c.head_stride;
    float qr[E], o[E], m = -INFINITY, l = 0.0f;
    for (int e = 0; e < E; ++e) { qr[e] = q[i * q_stride + h * HS + lane * E + e]; o[e] = 0.0f; }
    for (int t = w; t < len; t += WARPS) {
        const int page = tables[(size_t)i * max_pages + t / c.page_size];
        if (page < 0 || page >= c.pages) continue;
        const long long at = page * c.page_stride + (t % c.page_size) * c.token_stride + lane * E;
        float s = 0.0f;
        for (int e = 0; e < E; ++e) s = fmaf(qr[e], to_float(K[at + e]), s);
        s = warp_sum(s) * scale;
        const float mn = fmaxf(m, s), keep = expf(m - mn), p = expf(s - mn);
        l = l * keep + p;
        for (int e = 0; e < E; ++e) o[e] = fmaf(p, to_float(V[at + e]), o[e] * keep);
        m = mn;
    }
    if (lane == 0) { m_of[w] = m; l_of[w] = l; }
    for (int e = 0; e < E; ++e) o_of[w][lane * E + e] = o[e];
    __syncthreads();
    float top = -INFINITY, all = 0.0f;
    for (int j = 0; j < WARPS; ++j) top = fmaxf(top, m_of[j]);
    for (int j = 0; j < WARPS; ++j) all += l_of[j] > 0.0f ? l_of[j] * expf(m_of[j] - top) : l_of[j];
    for (int d = threadIdx.x; d < HS; d += blockDim.x) {
        float x = 0.0f;
        for (int j = 0; j < WARPS; ++j) if (l_of[j] != 0.0f) x += o_of[j][d] * expf(m_of[j] - top);
        out[i * out_stride + h * HS + d] = all == 0.0f ? 0.0f : x / all;
    }
    if (lse && threadIdx.x == 0) lse[(size_t)i * heads + h] = all == 0.0f ? -INFINITY : top + logf(all);
}

size_t element(int type) { return type == BMB_TYPE_FP32 ? 4 : 2; }

int check_cache(const char *what, const bmb_kv_cache *c) {
    if (!c || !c->k || !c->v) return fail(BMB_E_ARG, "%s: no cache", what);
    if (c->type < BMB_TYPE_FP32 || c->type > BMB_TYPE_FP16) return fail(BMB_E_ARG, "%s: unknown type %d", what, c->type);
    if (c->pages <= 0 || c->page_size <= 0 || c->heads <= 0)
        return fail(BMB_E_ARG, "%s: bad sizes (pages=%d page_size=%d heads=%d)", what, c->pages, c->page_size, c->heads);
    if (c->head_size != 32 && c->head_size != 64 && c->head_size != 128)
        return fail(BMB_E_UNSUPPORTED, "%s: head size %d (32, 64 and 128 are served)", what, c->head_size);
    if ((long long)c->pages * c->page_size > INT_MAX) return fail(BMB_E_LIMIT, "%s: %d pages of %d tokens are beyond an int", what, c->pages, c->page_size);
    const long long unit = 16 / (long long)element(c->type);
    const long long strides[] = {c->page_stride, c->token_stride, c->head_stride};
    for (long long s : strides)
        if (s < c->head_size || s % unit) return fail(BMB_E_ARG, "%s: stride %lld (multiples of 16 bytes, at least the head size)", what, s);
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return fail(BMB_E_ARG, "%s: the cache is not 16-byte aligned", what);
    return BMB_OK;
}

template <typename T>
int run_attend(float *out, float *lse, const float *q, const bmb_kv_cache &c, const int *tables, const int *lens, int n, int heads,
               long long q_stride, long long out_stride, int max_pages, float scale, cudaStream_t st) {
    switch (c.head_size) {
    case 32: return launch(false, attend_k<T, 32>, n * heads, 256, 0, st, out, lse, q, c, tables, lens, heads, q_stride, out_stride, max_pages, scale);
    case 64: return launch(false, attend_k<T, 64>, n * heads, 256, 0, st, out, lse, q, c, tables, lens, heads, q_stride, out_stride, max_pages, scale);
    default: return launch(false, attend_k<T, 128>, n * heads, 256, 0, st, out, lse, q, c, tables, lens, heads, q_stride, out_stride, max_pages, scale);
    }
}

}  // namespace
}  // namespace bmb

using namespace bmb;

extern "C" {

int bmb_paged_kv_write(const bmb_kv_cache *cache, const float *k, const float *v, long long row_stride, const int *slots, int tokens, void *stream) {
    BMB_TRY(check_cache("paged_kv_write", cache));
    if (tokens < 0 || row_stride < 0) return fail(BMB_E_ARG, "paged_kv_write: tokens=%d row_stride=%lld", tokens, row_stride);
    if (tokens == 0) return BMB_OK;
    if (!k || !v || !slots || ((uintptr_t)k | (uintptr_t)v) & 3) return fail(BMB_E_ARG, "paged_kv_write: a null or unaligned pointer");
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->type == BMB_TYPE_FP32) return launch(false, kv_write_k<float>, tokens, 256, 0, st, *cache, k, v, row_stride, slots);
    if (cache->type == BMB_TYPE_BF16) return launch(false, kv_write_k<__nv_bfloat16>, tokens, 256, 0, st, *cache, k, v, row_stride, slots);
    return launch(false, kv_write_k<__half>, tokens, 256, 0, st, *cache, k, v, row_stride, slots);
}

size_t bmb_paged_attention_workspace(int heads, int kv_heads, int head_size) {
    (void)heads; (void)kv_heads; (void)head_size;
    return 16;
}

int bmb_paged_attention(float *out, float *lse, const float *q, const bmb_kv_cache *cache, const int *tables, const int *lens, int n, int heads,
                        long long q_stride, long long out_stride, int max_pages, float scale, void *workspace, size_t workspace_bytes, void *stream) {
    BMB_TRY(check_cache("paged_attention", cache));
    if (n < 0 || heads <= 0 || heads % cache->heads || max_pages <= 0)
        return fail(BMB_E_ARG, "paged_attention: bad sizes (n=%d heads=%d, %d in the cache, max_pages=%d)", n, heads, cache->heads, max_pages);
    if (q_stride < 0 || out_stride < (long long)heads * cache->head_size)
        return fail(BMB_E_ARG, "paged_attention: q_stride=%lld out_stride=%lld", q_stride, out_stride);
    if ((long long)max_pages * cache->page_size > INT_MAX)
        return fail(BMB_E_LIMIT, "paged_attention: %d pages of %d tokens are beyond an int", max_pages, cache->page_size);
    if ((long long)n * heads > INT_MAX) return fail(BMB_E_LIMIT, "paged_attention: %d requests of %d heads", n, heads);
    if (n == 0) return BMB_OK;
    if (!out || !q || !tables || !lens || (((uintptr_t)out | (uintptr_t)q) & 3)) return fail(BMB_E_ARG, "paged_attention: a null or unaligned pointer");
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < bmb_paged_attention_workspace(heads, cache->heads, cache->head_size))
        return fail(BMB_E_ARG, "paged_attention: a workspace of %zu bytes, 16-byte aligned, is needed (got %zu)",
                    bmb_paged_attention_workspace(heads, cache->heads, cache->head_size), workspace_bytes);
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->type == BMB_TYPE_FP32)
        return run_attend<float>(out, lse, q, *cache, tables, lens, n, heads, q_stride, out_stride, max_pages, scale, st);
    if (cache->type == BMB_TYPE_BF16)
        return run_attend<__nv_bfloat16>(out, lse, q, *cache, tables, lens, n, heads, q_stride, out_stride, max_pages, scale, st);
    return run_attend<__half>(out, lse, q, *cache, tables, lens, n, heads, q_stride, out_stride, max_pages, scale, st);
}

}  // extern "C"
