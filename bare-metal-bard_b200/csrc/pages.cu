// Pages of a cache that several requests share: handed out by the requests' lengths (bmb_pages_assign) and taken back
// (bmb_pages_release), on the GPU, so that a step's shapes never have to come back to the host.
//
// Both are sums over requests in their order (where a request's tokens and pages begin) and stores that follow from them.  What they
// move is little, so what they take is the chain of loads: lengths, then pages.  A block counts a stretch of requests with a thread
// each, and tokens (of assign) or table entries (of release) are then dealt to threads whatever requests they are of.  Few
// of them: one block.  Many: a cluster of 8, each of which counts all requests and takes an eighth of the tokens or entries; lengths are
// read by all before any is overwritten, which a cluster's barrier can say and a grid cannot.
#include "common.cuh"
#include <atomic>
#include <climits>
#include <type_traits>

namespace bmb {
namespace {

constexpr int PG_CLUSTER = 8, PG_MOST = 1024, PG_STASH = 192 * 1024;
template <int V> using Int = std::integral_constant<int, V>;

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
template <int BLOCKS>
__device__ __forceinline__ void sync_all() {
    if (BLOCKS == 1) {
        __syncthreads();
    } else {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}
// *p of another block of the cluster
__device__ __forceinline__ long long read_of(const long long *p, unsigned rank) {
    long long v;
    asm volatile("{\n.reg .u32 a;\nmapa.shared::cluster.u32 a, %1, %2;\nld.shared::cluster.s64 %0, [a];\n}" : "=l"(v) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank) : "memory");
    return v;
}

// The sum over the threads before and including this one; `total`: of all of them.  `sums` (shared, one a warp) is free again after the
// next barrier.
template <int THREADS>
__device__ __forceinline__ long long block_scan(long long v, long long *sums, long long *total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) sums[w] = v;
    __syncthreads();
    long long s = lane < THREADS / 32 ? sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    *total = __shfl_sync(0xffffffffu, s, 31);
    const long long before = __shfl_sync(0xffffffffu, s, w > 0 ? w - 1 : 0);
    return v + (w > 0 ? before : 0);
}

__device__ __forceinline__ int pages_of(int tokens, int page_size) { return (int)(((long long)tokens + page_size - 1) / page_size); }

template <int BLOCKS, int THREADS>
__global__ void __launch_bounds__(THREADS) assign_k(int *tables, int *lens_out, int *slots, int *positions, int *owners, int *starts,
                                                    int *free_left, const int *lens, const int *new_lens, const int *free_pages,
                                                    const int *free_count, int n, int max_pages, int page_size, int pages, int max_tokens) {
    __shared__ long long sums[2][THREADS / 32];
    // of the stretch's requests: where tokens and new pages begin, length, pages held (< 0: not served, ~held)
    __shared__ int begin_of[THREADS], page_begin[THREADS], len_of[THREADS], held_of[THREADS];
    __shared__ int taken;
    const int me = BLOCKS == 1 ? 0 : (int)cluster_rank();
    if (threadIdx.x == 0) taken = 0;
    let_successor_start();
    wait_for_predecessor();
    const int F = min(max(*free_count, 0), pages);
    long long tokens_before = 0, pages_before = 0;
    for (int base = 0; base < n; base += THREADS) {
        const int i = base + threadIdx.x;
        const int L = i < n ? max(lens[i], 0) : 0, A = i < n ? max(new_lens[i], 0) : 0;
        long long all;
        const long long end = tokens_before + block_scan<THREADS>(A, sums[0], &all);
        const int chunk_begin = (int)min(tokens_before, (long long)max_tokens);
        tokens_before += all;
        const int chunk_end = (int)min(tokens_before, (long long)max_tokens);
        const int held = pages_of(L, page_size);
        const long long want = ((long long)L + A + page_size - 1) / page_size;
        const bool fits = i < n && want <= max_pages && end <= max_tokens;
        const int need = fits ? (int)want - held : 0;
        const long long last = pages_before + block_scan<THREADS>(need, sums[1], &all);
        pages_before += all;
        const bool served = fits && (need == 0 || last <= F);
        begin_of[threadIdx.x] = i < n ? (int)min(end - A, (long long)max_tokens) : INT_MAX;
        page_begin[threadIdx.x] = served ? (int)(last - need) : 0;
        len_of[threadIdx.x] = L;
        held_of[threadIdx.x] = served ? held : ~held;
        if (served && need > 0) atomicMax(&taken, (int)last);
        sync_all<BLOCKS>();                                   // the arrays are filled, and all blocks have read these lengths
        if (me == 0 && i < n) {
            lens_out[i] = served ? L + A : L;
            if (starts) starts[i] = begin_of[threadIdx.x];
        }
        // (unsigned: the last step may end behind an int, by no more than a stretch)
        for (unsigned next = (unsigned)chunk_begin + me * THREADS + threadIdx.x; next < (unsigned)chunk_end; next += BLOCKS * THREADS) {
            const int t = (int)next;
            int r = 0;                                        // the last request that begins at t or before it
#pragma unroll
            for (int step = THREADS / 2; step > 0; step >>= 1)
                if (begin_of[r + step] <= t) r += step;
            const long long at = (long long)len_of[r] + (t - begin_of[r]);
            const int pos = (int)min(at, (long long)INT_MAX), held_r = held_of[r];
            int slot = -1;
            if (held_r >= 0) {
                const int k = pos / page_size, off = pos - k * page_size;
                int *entry = tables + (size_t)(base + r) * max_pages + k;
                int page;
                if (k >= held_r) {
                    page = free_pages[F - 1 - (page_begin[r] + k - held_r)];
                    if (off == 0) *entry = page;              // (a new page begins with a new token)
                } else {
                    page = *entry;
                }
                if (page >= 0 && page < pages) slot = page * page_size + off;
            }
            slots[t] = slot;
            if (positions) positions[t] = pos;
            if (owners) owners[t] = base + r;
        }
        __syncthreads();
    }
    for (long long t = tokens_before + me * THREADS + threadIdx.x; t < max_tokens; t += BLOCKS * THREADS) {
        slots[t] = -1;
        if (positions) positions[t] = 0;
        if (owners) owners[t] = -1;
    }
    sync_all<BLOCKS>();                                       // (all have read free_count, if there was no request)
    if (me == 0 && threadIdx.x == 0) {
        *free_left = F - taken;
        if (starts) starts[n] = (int)min(tokens_before, (long long)max_tokens);
    }
}

template <int BLOCKS, int THREADS>
__global__ void __launch_bounds__(THREADS) release_k(int *free_pages, int *free_out, int *lens_out, const int *free_count, const int *lens,
                                                     const int *tables, const int *done, int n, int max_pages, int page_size, int pages, int stash) {
    extern __shared__ int stashed[];                          // [warps][stash]: a warp's entries, if it has no more than that
    __shared__ long long sums[2][THREADS / 32];
    __shared__ long long end_of[THREADS];                     // where the entries of the stretch's requests end
    __shared__ long long found;                               // pages of the pool among this block's entries
    const int me = BLOCKS == 1 ? 0 : (int)cluster_rank(), lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    let_successor_start();
    wait_for_predecessor();
    const int F = min(max(*free_count, 0), pages);
    long long before = F;
    for (int base = 0; base < n; base += THREADS) {
        const int i = base + threadIdx.x;
        const bool ends = i < n && done[i] != 0;
        const int L = i < n ? max(lens[i], 0) : 0;
        long long entries, all;
        end_of[threadIdx.x] = block_scan<THREADS>(ends ? min(pages_of(L, page_size), max_pages) : 0, sums[0], &entries);
        sync_all<BLOCKS>();                                   // as in assign_k
        if (me == 0 && i < n) lens_out[i] = ends ? 0 : L;
        // A run of entries for each warp, in order; once to count and once to write, the second time from shared memory where there is room
        // (100 thousand entries read twice: 13.2 us, once: 10.7).
        constexpr int WARPS = BLOCKS * THREADS / 32, AHEAD = 4;
        const long long each = (entries + WARPS * 32 - 1) / (WARPS * 32) * 32;
        const long long from = (me * (THREADS / 32) + w) * each, to = min(from + each, entries);
        const bool kept = each <= stash;
        int *mine_stashed = stashed + w * stash;
        auto read = [&](auto &&use) {
            int r = 0;
            for (long long f = from + lane; f - lane < to; f += 32 * AHEAD) {
                int page[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const long long e = f + 32 * k;
                    page[k] = -1;
                    if (e < to) {
                        // the first request that ends behind e: one of the next, or far on
                        for (int i = 0; i < 4 && end_of[r] <= e; ++i) ++r;
                        if (end_of[r] <= e) {
                            r = 0;
#pragma unroll
                            for (int step = THREADS / 2; step > 0; step >>= 1)
                                if (end_of[r + step - 1] <= e) r += step;
                        }
                        page[k] = tables[(size_t)(base + r) * max_pages + (e - (r > 0 ? end_of[r - 1] : 0))];
                    }
                }
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    if (kept && f + 32 * k < to) mine_stashed[f + 32 * k - from] = page[k];
                    use(page[k]);
                }
            }
        };
        int mine = 0;
        read([&](int page) { mine += __popc(__ballot_sync(0xffffffffu, (unsigned)page < (unsigned)pages)); });
        long long at = block_scan<THREADS>(lane == 31 ? mine : 0, sums[1], &all) - (lane == 31 ? mine : 0);
        at = before + __shfl_sync(0xffffffffu, at, 31);
        if (BLOCKS > 1) {
            if (threadIdx.x == 0) found = all;
            sync_all<BLOCKS>();
            all = 0;
            for (int b = 0; b < BLOCKS; ++b) {
                const long long x = read_of(&found, b);
                all += x;
                if (b < me) at += x;
            }
        }
        auto write = [&](int page) {
            const unsigned ok = __ballot_sync(0xffffffffu, (unsigned)page < (unsigned)pages);
            const long long place = at + __popc(ok & ((1u << lane) - 1));
            if ((ok >> lane & 1) && place < pages) free_pages[place] = page;
            at += __popc(ok);
        };
        if (kept) {
            const int count = (int)max(to - from, 0LL);
            for (int i = lane; i - lane < count; i += 32) write(i < count ? mine_stashed[i] : -1);
        } else {
            read(write);
        }
        before += all;
        sync_all<BLOCKS>();                                   // (the others have read `found`)
    }
    if (n == 0) sync_all<BLOCKS>();
    if (me == 0 && threadIdx.x == 0) *free_out = (int)min(before, (long long)pages);
}

// Up to 256 requests and 1024 tokens (or table entries, by the tables' size): one block of 256 threads.  Up to 2048 tokens or 8192 entries: one of
// 1024.  Beyond: a cluster of 8.  Measured, us: 64 tokens 3.0 with 256 threads, 3.9 with 1024; 1424 tokens of 256 requests 5.9, 5.0 and
// 5.3 with the cluster; 15 thousand tokens 15.7 with 1024, 6.0 with the cluster.  Release (its entries
// read twice) from tables of 1024 entries 4.2 and 4.2; of 4000 7.3, 5.3 and 7.2; of 62 thousand 13.5 with 1024 and 7.9 with the cluster.
constexpr int PG_FEW_REQUESTS = 256, PG_FEW = 1024, PG_SOME_TOKENS = 2048, PG_SOME_ENTRIES = 8192;

int check_pool(const char *what, int n, int max_pages, int page_size, int pages) {
    if (n < 0 || max_pages <= 0 || page_size <= 0 || pages < 0)
        return fail(BMB_E_ARG, "%s: bad sizes (n=%d max_pages=%d page_size=%d pages=%d)", what, n, max_pages, page_size, pages);
    if (n > INT_MAX - (PG_MOST - 1)) return fail(BMB_E_LIMIT, "%s: %d requests", what, n);      // (the first one behind the last stretch is an int)
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
    if (!words(tables, lens_out, slots, positions, owners, starts, free_left, lens, new_lens, free_pages, free_count))
        return fail(BMB_E_ARG, "pages_assign: an unaligned pointer");
    auto run = [&](auto blocks, auto threads) {
        constexpr int B = decltype(blocks)::value, N = decltype(threads)::value;
        return launch_cluster(assign_k<B, N>, B, B, N, 0, (cudaStream_t)stream, tables, lens_out, slots, positions, owners, starts, free_left, lens, new_lens,
                                 free_pages, free_count, n, max_pages, page_size, pages, max_tokens);
    };
    if (n <= PG_FEW_REQUESTS && max_tokens <= PG_FEW) return run(Int<1>(), Int<256>());
    return max_tokens <= PG_SOME_TOKENS ? run(Int<1>(), Int<PG_MOST>()) : run(Int<PG_CLUSTER>(), Int<PG_MOST>());
}

int bmb_pages_release(int *free_pages, int *free_out, int *lens_out, const int *free_count, const int *lens, const int *tables, const int *done,
                      int n, int max_pages, int page_size, int pages, void *stream) {
    BMB_TRY(check_pool("pages_release", n, max_pages, page_size, pages));
    if (!free_out || !free_count || (pages && !free_pages) || (n && (!tables || !lens_out || !lens || !done)))
        return fail(BMB_E_ARG, "pages_release: a null pointer");
    if (!words(free_pages, free_out, lens_out, free_count, lens, tables, done)) return fail(BMB_E_ARG, "pages_release: an unaligned pointer");
    const long long entries = (long long)n * max_pages;
    auto run = [&](auto blocks, auto threads) -> int {
        constexpr int B = decltype(blocks)::value, N = decltype(threads)::value, MOST = PG_STASH / (N / 32) / 4;
        // what a warp may have at most, if that fits
        const long long each = (entries + B * N - 1) / (B * N) * 32;
        const int stash = each <= MOST ? (int)each : 0;
        static std::atomic<unsigned long long> prepared{0};       // devices (those from 64 on are prepared every time)
        const int dev = current_device();
        const unsigned long long bit = dev >= 0 && dev < 64 ? 1ULL << dev : 0;
        if (!(prepared.load(std::memory_order_relaxed) & bit)) {
            BMB_CUDA(cudaFuncSetAttribute(release_k<B, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, PG_STASH));
            prepared.fetch_or(bit, std::memory_order_relaxed);
        }
        return launch_cluster(release_k<B, N>, B, B, N, (size_t)stash * (N / 32) * sizeof(int), (cudaStream_t)stream, free_pages, free_out, lens_out, free_count,
                              lens, tables, done, n, max_pages, page_size, pages, stash);
    };
    if (n <= PG_FEW_REQUESTS && entries <= PG_FEW) return run(Int<1>(), Int<256>());
    return entries <= PG_SOME_ENTRIES ? run(Int<1>(), Int<PG_MOST>()) : run(Int<PG_CLUSTER>(), Int<PG_MOST>());
}

}  // extern "C"
