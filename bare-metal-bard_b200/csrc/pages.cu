// Pages of a cache that several requests share: handed out by the requests' lengths (bmb_pages_assign) and taken back
// (bmb_pages_release), on the GPU, so that a step's shapes never have to come back to the host.
//
// Both are sums over requests in their order (where a request's tokens and pages begin) and stores that follow from them.
#include "common.cuh"
#include <climits>

namespace bmb {
namespace {

constexpr int PG_THREADS = 1024, PG_WARPS = PG_THREADS / 32;

// The sum over the threads before and including this one; `total`: of all of them. `warps` is shared.
__device__ __forceinline__ long long block_scan(long long v, long long *warps, long long *total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) warps[w] = v;
    __syncthreads();
    long long before = 0, all = 0;
    for (int i = 0; i < PG_WARPS; ++i) {
        if (i < w) before += warps[i];
        all += warps[i];
    }
    *total = all;
    return before + v;
}

__device__ __forceinline__ int pages_of(long long tokens, int page_size) { return (int)((tokens + page_size - 1) / page_size); }

__global__ void __launch_bounds__(PG_THREADS) assign_k(int *tables, int *lens_out, int *slots, int *positions, int *owners, int *starts,
                                                       int *free_left, const int *lens, const int *new_lens, const int *free_pages,
                                                       const int *free_count, int n, int max_pages, int page_size, int pages, int max_tokens) {
    __shared__ long long warps[PG_WARPS];
    __shared__ long long begin_of[PG_THREADS], page_begin[PG_THREADS];
    __shared__ int len_of[PG_THREADS], new_of[PG_THREADS], need_of[PG_THREADS];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int F = min(max(*free_count, 0), pages);
    long long tokens_before = 0, pages_before = 0, taken = 0;
    for (int base = 0; base < n; base += PG_THREADS) {
        const int i = base + threadIdx.x;
        const int L = i < n ? max(lens[i], 0) : 0, A = i < n ? max(new_lens[i], 0) : 0;
        long long all;
        const long long end = tokens_before + block_scan(A, warps, &all);
        tokens_before += all;
        const long long want = (L + (long long)A + page_size - 1) / page_size;
        const bool fits = i < n && want <= max_pages && end <= max_tokens;
        const int need = fits ? (int)want - pages_of(L, page_size) : 0;
        const long long last = pages_before + block_scan(need, warps, &all);
        pages_before += all;
        const bool served = fits && (need == 0 || last <= F);
        begin_of[threadIdx.x] = end - A;
        page_begin[threadIdx.x] = last - need;
        len_of[threadIdx.x] = L;
        new_of[threadIdx.x] = A;
        need_of[threadIdx.x] = served ? need : -1;
        if (i < n) {
            lens_out[i] = served ? L + A : L;
            if (starts) starts[i] = (int)min(end - A, (long long)max_tokens);
        }
        (void)block_scan(served ? need : 0, warps, &all);
        taken += all;                    // (its barriers also publish the arrays)
        for (int r = w; r < min(PG_THREADS, n - base); r += PG_WARPS) {
            const long long S = begin_of[r];
            const int Lr = len_of[r], Ar = new_of[r], needed = need_of[r];
            int *table = tables + (size_t)(base + r) * max_pages;
            const int have = pages_of(Lr, page_size);
            for (int k = lane; k < needed; k += 32) table[have + k] = free_pages[F - 1 - (int)(page_begin[r] + k)];
            __syncwarp();
            for (int j = lane; j < Ar && S + j < max_tokens; j += 32) {
                const int at = (int)S + j, pos = (int)min((long long)Lr + j, (long long)INT_MAX);
                int slot = -1;
                if (needed >= 0) {
                    const int page = table[pos / page_size];
                    if (page >= 0 && page < pages) slot = page * page_size + pos % page_size;
                }
                slots[at] = slot;
                if (positions) positions[at] = pos;
                if (owners) owners[at] = base + r;
            }
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        *free_left = F - (int)taken;
        if (starts) starts[n] = (int)min(tokens_before, (long long)max_tokens);
    }
    for (long long t = tokens_before + threadIdx.x; t < max_tokens; t += PG_THREADS) {
        slots[t] = -1;
        if (positions) positions[t] = 0;
        if (owners) owners[t] = -1;
    }
}

__global__ void __launch_bounds__(PG_THREADS) release_k(int *free_pages, int *free_out, int *lens_out, const int *free_count, const int *lens,
                                                        const int *tables, const int *done, int n, int max_pages, int page_size, int pages) {
    __shared__ long long warps[PG_WARPS];
    __shared__ long long begin_of[PG_THREADS];
    __shared__ int held[PG_THREADS], valid[PG_THREADS];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int F = min(max(*free_count, 0), pages);
    long long before = F;
    for (int base = 0; base < n; base += PG_THREADS) {
        const int i = base + threadIdx.x;
        const bool ends = i < n && done[i] != 0;
        const int L = i < n ? max(lens[i], 0) : 0;
        held[threadIdx.x] = ends ? min(pages_of(L, page_size), max_pages) : 0;
        if (i < n) lens_out[i] = ends ? 0 : L;
        __syncthreads();
        for (int r = w; r < PG_THREADS; r += PG_WARPS) {
            const int *table = tables + (size_t)min(base + r, n - 1) * max_pages;
            int count = 0;
            for (int k = 0; k < held[r]; k += 32) {
                const int page = k + lane < held[r] ? table[k + lane] : -1;
                count += __popc(__ballot_sync(0xffffffffu, page >= 0 && page < pages));
            }
            if (lane == 0) valid[r] = count;
        }
        __syncthreads();
        long long all;
        const int mine = valid[threadIdx.x];
        begin_of[threadIdx.x] = before + block_scan(mine, warps, &all) - mine;
        before += all;
        __syncthreads();
        for (int r = w; r < PG_THREADS; r += PG_WARPS) {
            const int *table = tables + (size_t)min(base + r, n - 1) * max_pages;
            long long at = begin_of[r];
            for (int k = 0; k < held[r]; k += 32) {
                const int page = k + lane < held[r] ? table[k + lane] : -1;
                const unsigned ok = __ballot_sync(0xffffffffu, page >= 0 && page < pages);
                const long long to = at + __popc(ok & ((1u << lane) - 1));
                if ((ok >> lane & 1) && to < pages) free_pages[to] = page;
                at += __popc(ok);
            }
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) *free_out = (int)min(before, (long long)pages);
}

int check_pool(const char *what, int n, int max_pages, int page_size, int pages) {
    if (n < 0 || max_pages <= 0 || page_size <= 0 || pages < 0)
        return fail(BMB_E_ARG, "%s: bad sizes (n=%d max_pages=%d page_size=%d pages=%d)", what, n, max_pages, page_size, pages);
    if ((long long)pages * page_size > INT_MAX || (long long)max_pages * page_size > INT_MAX)
        return fail(BMB_E_LIMIT, "%s: %d (a row of the tables: %d) pages of %d tokens are beyond an int", what, pages, max_pages, page_size);
    return BMB_OK;
}

}  // namespace
}  // namespace bmb

using namespace bmb;

extern "C" {

int bmb_pages_assign(int *tables, int *lens_out, int *slots, int *positions, int *owners, int *starts, int *free_left, const int *lens,
                     const int *new_lens, const int *free_pages, const int *free_count, int n, int max_pages, int page_size, int pages,
                     int max_tokens, void *stream) {
    BMB_TRY(check_pool("pages_assign", n, max_pages, page_size, pages));
    if (max_tokens < 0) return fail(BMB_E_ARG, "pages_assign: max_tokens=%d", max_tokens);
    if (!free_left || !free_count || (pages && !free_pages) || (max_tokens && !slots) || (n && (!tables || !lens_out || !lens || !new_lens)))
        return fail(BMB_E_ARG, "pages_assign: a null pointer");
    return launch(false, assign_k, 1, PG_THREADS, 0, (cudaStream_t)stream, tables, lens_out, slots, positions, owners, starts, free_left, lens,
                  new_lens, free_pages, free_count, n, max_pages, page_size, pages, max_tokens);
}

int bmb_pages_release(int *free_pages, int *free_out, int *lens_out, const int *free_count, const int *lens, const int *tables, const int *done,
                      int n, int max_pages, int page_size, int pages, void *stream) {
    BMB_TRY(check_pool("pages_release", n, max_pages, page_size, pages));
    if (!free_out || !free_count || (pages && !free_pages) || (n && (!tables || !lens_out || !lens || !done)))
        return fail(BMB_E_ARG, "pages_release: a null pointer");
    return launch(false, release_k, 1, PG_THREADS, 0, (cudaStream_t)stream, free_pages, free_out, lens_out, free_count, lens, tables, done, n,
                  max_pages, page_size, pages);
}

}  // extern "C"
