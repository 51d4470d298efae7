// A paged cache of keys and values, and attention of one new token of each request over its pages.
#include "flash_mma.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>
#include <vector>

namespace bmb {
namespace {

__host__ __device__ inline long long div_near(long long a, int b) { return a >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b); }

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Keys and values of new tokens into their slots: a thread takes 16 bytes of the cache, of keys and of values.  Bound by memory.  VEC: the
// rows are 16-byte aligned.
constexpr int KW_THREADS = 256;
template <typename T, bool VEC>
__global__ void __launch_bounds__(KW_THREADS) kv_write_k(const __grid_constant__ bmb_kv_cache c, const float *k, const float *v, long long row_stride, const int *slots,
                                                         int tokens, int units) {
    constexpr int E = 16 / (int)sizeof(T);                    // elements a unit; `units` of them a row
    let_successor_start();
    wait_for_predecessor();
    const long long at = (long long)blockIdx.x * KW_THREADS + threadIdx.x;
    if (at >= (long long)tokens * units) return;              // (before the division: its result is an int)
    const int token = (int)div_near(at, units), e = (int)(at - (long long)token * units) * E;
    const int slot = slots[token];
    float x[2][E];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float *from = (i ? v : k) + token * row_stride + e;
#pragma unroll
        for (int j = 0; j < E; j += VEC ? 4 : 1) {
            if (VEC) *reinterpret_cast<float4 *>(&x[i][j]) = *reinterpret_cast<const float4 *>(from + j);
            else x[i][j] = from[j];
        }
    }
    if (slot < 0 || slot >= c.pages * c.page_size) return;
    const int page = slot / c.page_size, head = e / c.head_size;
    const long long to = page * c.page_stride + (slot - page * c.page_size) * c.token_stride + head * c.head_stride + (e - head * c.head_size);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        alignas(16) T y[E];
#pragma unroll
        for (int j = 0; j < E; ++j) y[j] = from_float<T>(x[i][j]);
        *reinterpret_cast<uint4 *>((T *)(i ? c.v : c.k) + to) = *reinterpret_cast<const uint4 *>(y);
    }
}

template <typename T>
int run_write(const bmb_kv_cache &c, const float *k, const float *v, long long row_stride, const int *slots, int tokens, cudaStream_t st) {
    const int units = c.heads * c.head_size / (16 / (int)sizeof(T));
    const long long blocks = ((long long)tokens * units + KW_THREADS - 1) / KW_THREADS;
    if (blocks > INT_MAX) return fail(BMB_E_LIMIT, "paged_kv_write: %d tokens of %d heads", tokens, c.heads);
    const bool vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && row_stride % 4 == 0;
    return launch_in_chain(vec ? kv_write_k<T, true> : kv_write_k<T, false>, (unsigned)blocks, KW_THREADS, 0, st, c, k, v, row_stride, slots, tokens, units);
}

// ---- attention of one token of each request ---------------------------------------------------------------------------
//
// out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q . k_j, with running m, sums and outputs in one pass over keys and
// values, which is all the work there is: 2 to 4 operations a byte for each query head that shares them.  So what counts is that the
// loads never pause, on every SM alike, whatever the lengths are.
//
// Work: the tiles of all requests and cache heads stand in one line, a tile being 4 KB of keys and 4 KB of values, and are cut
// into equal runs, one for each warp of the GPU.  A warp is on its own: its tiles come by cp.async through a ring of its own, over the
// borders of heads and requests, and no block-wide barrier stands in the loop.  Heads that lie in several runs are joined, first
// among the warps of a block, and what reaches over blocks by attend_join_k.  Few or short heads go to a cluster of blocks each instead
// (blocks_alone).  Nothing depends on arrival, so equal calls give equal bits.
//
// Arithmetic: warp-level matrix instructions, 8 query heads of one cache head a time, at fp32 accuracy.  Queries and weights are
// fp32, so each goes in as pieces of the cache's type, whose products with its elements are exact: the 16 rows of an
// instruction are the 8 rows' first pieces and their second ones, so a row's two sums lie in one lane and are added there.  fp16:
// two pieces of 11 bits, scaled by a power of two for each row of q (weights by 2^14), kept down to 2^-38 of the row's
// largest.  bf16: three of 8 bits, the third in an instruction of its own.  fp32: two TF32 pieces (fm, flash_mma.cuh) of queries and
// weights, and of keys and values as they are read (cutting the first piece off instead of rounding it saved 1 % and lost a bit: errors of
// 4.5e-7 in the 2-norm for 2.8e-7).  Sums over tiles are kept in fp32 registers.  Masked and absent tokens are zeros in
// shared memory with a weight of zero, whatever the memory there holds.
//
// Pieces of an infinity, and of an fp32 element within 2^-12 of the largest number, whose first piece is rounded to one, cancel to NaN where the formula
// has an infinity or a finite result.  A score of NaN, and an infinity or NaN in a sum of values, is still there when a head ends; what lost its sign would
// be NaN too, so sums that are finite are right.  A warp that had others works on those heads (its parts of them) once more when its run is
// done, a token at a time in plain fp32: what it leaves is what the formula gives.  The check at a head's end and the code for it cost
// up to 0.1 us of the 6.2 of one text of 256 tokens, up to 0.3 of 15.3 where heads end with nearly every tile, and up to 0.5 % of 100.
//
// Bound by, and measured (us, caches cold): 609 MB of fp16, 8 requests of up to 32768 tokens, 32 heads on 8 of 128: 100, 6.1 TB/s, the loads.  203 MB of
// fp32, 37 of up to 2777, 16 heads on 4 of 128: 44.5, and 101 MB of bf16, 64 of up to 1024, 12 heads of 64: 26.8: the loads alone take 40.8 and
// 24.6 of that, at 6.2 TB/s behind 4 us before the first tile is there and in front of 4 for the last warps and the joins; the arithmetic alone 43.3
// and 24.5 (8 warps an SM, issue slots 43 and 34 % in use; with 12 warps and shorter rings 1 to 4 us more in all).
constexpr int PA_WARPS = 4, PA_THREADS = 32 * PA_WARPS, PA_STAGES = 3, PA_TILE = 4096, PA_ROWS = 8;
constexpr int PA_BLOCKS = 2, PA_MOST_BLOCKS = 512;          // blocks an SM, and in all
constexpr size_t PA_SMEM = 112 * 1024;                       // dynamic shared memory with which two blocks fit an SM
constexpr int PA_CLUSTER = 8;
constexpr float LOWEST = -3.402823466e38f;                   // the lowest number of fp32

// Blocks for each head, a cluster of them, or 0 for the line (below).  Where heads are few or short a cluster takes each alone: no line to find a
// place in and no second launch, which together are 2 to 4 us of GPU time and 4 of the host's.  But then the longest head alone says how long it
// takes, 0.7 us for each tile that a warp has of it, where the line spreads over all SMs.  As many blocks a head as fill the GPU (7/8 of the blocks that
// it holds: clusters do not fill its last ones) and have a tile for each warp; and then no more tiles a warp than 2, or 8 where the blocks fill the GPU.
// Measured, clusters / line, us, every length the longest that the tables hold: 6 heads of 64 fp32 (48 blocks) of 1, 2 and 4 tiles a warp 6.1 / 8.0,
// 7.4 / 8.1, 10.2 / 8.5; 48 heads bf16 (192) of 2, 4 and 8 tiles 7.8 / 10.0, 10.7 / 11.8, 17.1 / 18.3; 32 heads of 128 fp16 (256) of 2, 4 and 8 tiles
// 9.1 / 11.6, 11.6 / 15.1, 17.2 / 21.1; 288 heads bf16 of 4 and 8 tiles 11.3 / 15.9, 17.3 / 22.0.  With lengths from 1 up the line gains: 192 blocks
// of 8 tiles 13.2 / 11.6, 288 blocks of 8 tiles 16.0 / 16.3.
inline int blocks_alone(long long heads, int tiles, int blocks) {
    int k = 1;
    while (k < PA_CLUSTER && heads * 2 * k <= blocks * 7 / 8 && PA_WARPS * k < tiles) k *= 2;
    const int each = (tiles + PA_WARPS * k - 1) / (PA_WARPS * k);
    return heads * k <= blocks && each * (long long)blocks <= 2 * blocks + 6 * heads * k ? k : 0;
}

// All places in a line: requests in order, of each its (virtual) heads, of each its tiles and one place more, without work of its own, for
// what a head costs to begin and to end (without it the runs with many short heads were the last to end: 9 heads in one of 11 tiles
// took 31 us where the others took 24).
struct Line {
    long long places, each; // runs: warp w has places [begin(w), begin(w + 1)), `each` or one more
    int warps, rest;
    __host__ __device__ Line(long long places_, int most) : places(places_), warps((int)(places_ < most ? places_ > 1 ? places_ : 1 : most)) {
        each = div_near(places, warps);
        rest = (int)(places - each * warps);
    }
    __host__ __device__ long long begin(int w) const { return w * each + (w < rest ? w : rest); }
    __host__ __device__ int warp_of(long long place) const {
        const long long longer = rest * (each + 1);
        return (int)(place < longer ? place / (each + 1) : rest + (place - longer) / each);
    }
};
struct Shape {
    int n, heads, group, parts, vheads, cap, keys_log2;   // query heads a cache head, its groups of 8, virtual heads in all, longest length, keys a tile
    __host__ __device__ int length(int len) const { return len < 0 ? 0 : len < cap ? len : cap; }
    __host__ __device__ int stretch() const { return (n - 1) / PA_THREADS + 1; }       // requests that a thread counts the tiles of
    __host__ __device__ int places(int len) const { const int t = tiles(len); return t + (t > 0); }
    __host__ __device__ int tiles(int len) const { return (int)(((unsigned)length(len) + (1u << keys_log2) - 1) >> keys_log2); }
};
// A tile, and the request and virtual head that it is of.
struct Place {
    int request, vhead, tile, tiles, len;
    // To the tile at the place `in` behind the first one of request r, or behind that place if it has none.  Places passed over (0 or 1).
    __host__ __device__ int set(const Shape &s, const int *lens, int r, long long in) {
        for (; r + 1 < s.n && in >= (long long)s.places(lens[r]) * s.vheads; ++r) in -= (long long)s.places(lens[r]) * s.vheads;
        request = r;
        len = s.length(lens[r]);
        tiles = s.tiles(len);
        vhead = (int)div_near(in, tiles + 1);
        tile = (int)(in - (long long)vhead * (tiles + 1));
        if (tile < tiles) return 0;
        next_head(s, lens);
        return 1;
    }
    // (on the device a warp's lanes together: 32 requests without tokens are passed over at a time)
    __host__ __device__ void next_head(const Shape &s, const int *lens) {
        tile = 0;
        if (++vhead < s.vheads) return;
        vhead = tiles = 0;
#ifdef __CUDA_ARCH__
        const int lane = threadIdx.x & 31;
        for (++request; request < s.n; request += 32) {
            const int its = lane < s.n - request ? s.length(lens[request + lane]) : 0;
            const unsigned some = __ballot_sync(0xffffffffu, its > 0);
            if (some) {
                len = __shfl_sync(0xffffffffu, its, __ffs(some) - 1);
                request += __ffs(some) - 1;
                tiles = s.tiles(len);
                return;
            }
        }
#else
        while (tiles == 0 && ++request < s.n) {
            len = s.length(lens[request]);
            tiles = s.tiles(len);
        }
#endif
    }
    // places from this tile to the next, and the way there
    __host__ __device__ int step() const { return tile + 1 < tiles ? 1 : 2; }
    __host__ __device__ void next(const Shape &s, const int *lens) {
        if (++tile >= tiles) next_head(s, lens);
    }
};

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], const float (&a)[4], float b0, float b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])), "r"(__float_as_uint(a[3])),
                   "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
// 2^x by the special-function unit, results below 2^-126 as 0 (exp2f's steps to keep those are 3 instructions more).
__device__ __forceinline__ float two_to(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long x, y, z;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(z) : "l"(x), "l"(y));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(z));
    return a;
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __half) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ float2 unpack(uint32_t v, __half) { return __half22float2(*reinterpret_cast<__half2 *>(&v)); }
// A pair of fp32 values as pairs of pieces, the nearest value of the type each (bf16, three pieces: 8 bits each, cut off, which add up exactly);
// `pieces` of them.
template <typename T, int pieces>
__device__ __forceinline__ void split(float x, float y, uint32_t (&out)[pieces]) {
    if constexpr (pieces == 3) {
        float2 v = make_float2(x, y);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            out[i] = __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x7632);
            if (i < 2) v = add2(v, make_float2(-__uint_as_float(__float_as_uint(v.x) & 0xffff0000u), -__uint_as_float(__float_as_uint(v.y) & 0xffff0000u)));
        }
    } else {
#pragma unroll
        for (int i = 0; i < pieces; ++i) {
            out[i] = pack(x, y, T());
            const float2 v = unpack(out[i], T());
            x -= v.x;
            y -= v.y;
        }
    }
}

// n / d for 0 <= n < 2^31 and one d, by the method of Granlund and Montgomery (Division by invariant integers using multiplication, 1994): the
// high half of n times ceil(2^(32 + bits) / d) - 2^32, bits such that 2^bits >= d.  (The division of unknown numbers takes 20 instructions.)
struct Divide {
    unsigned by, mul, bits;
    Divide() = default;
    explicit Divide(unsigned d) : by(d), bits(0) {
        while (bits < 31 && (1u << bits) < d) ++bits;
        mul = (unsigned)(((1ULL << 32) * ((1ULL << bits) - d)) / d + 1);
    }
    __device__ __forceinline__ unsigned quotient(unsigned n) const { return (unsigned)(((unsigned long long)__umulhi(n, mul) + n) >> bits); }
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// *p of another block of the cluster
template <typename V>
__device__ __forceinline__ V read_of(const float *p, unsigned rank) {
    uint32_t a;
    V v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    if constexpr (sizeof(V) == 16) asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    else asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// Rows of a head in the workspace: of a block, the part of the head that it ends (0) and of the one that it begins (1).
struct Parts {
    float *o, *m, *l;      // [blocks][2][PA_ROWS][HS], [blocks][2][PA_ROWS]
    int4 *begun;           // [blocks]: request, virtual head, last block, 1; or w = 0 where the block begins no head that others go on with
};
constexpr size_t part_floats(int blocks, int hs) { return (size_t)blocks * 2 * PA_ROWS * (hs + 2); }
int attend_blocks() { return sm_count() * PA_BLOCKS < PA_MOST_BLOCKS ? sm_count() * PA_BLOCKS : PA_MOST_BLOCKS; }
size_t attend_workspace(int blocks, int hs) { return (part_floats(blocks, hs) * sizeof(float) + 15) / 16 * 16 + (size_t)blocks * sizeof(int4); }

struct Attend {
    float *out, *lse;
    const float *q;
    bmb_kv_cache c;
    const int *tables, *lens;
    long long q_stride, out_stride;
    int max_pages;
    Divide page_size;
    float scale;
    bool staged, aligned_q;      // queries are staged in shared memory, 16 bytes at a time
    int alone;                   // blocks for each head, a cluster (0: the line)
    Shape s;
    Parts w;
};

// A block's static shared memory.
struct AttendShared {
    float weight[2 * PA_WARPS][PA_ROWS];                                         // (aligned; and at the start:)
    struct RunBegin { long long in; int request; };                              // `in` places behind the first one of this request
    int4 part_of[PA_WARPS][2];                                                   // request, virtual head, 1 begins + 2 ends there, 1 (0: none)
    long long warp_total[PA_WARPS];                                              // (at the start)
    float part_m[PA_WARPS][2][PA_ROWS], part_l[PA_WARPS][2][PA_ROWS];
    int last_block[PA_WARPS + 1];                                                // that has a part of the head a warp has begun and not ended
};
static_assert(sizeof(AttendShared::weight) >= PA_WARPS * sizeof(AttendShared::RunBegin), "");
// Two blocks an SM: of its 228 KB each takes 1 KB beside its own, of which the static part is padded to the dynamic one's boundary.
static_assert(PA_BLOCKS * (PA_SMEM + 1024 + (sizeof(AttendShared) + 127) / 128 * 128) <= 228 * 1024, "");

template <typename T, int HS>
__global__ void __launch_bounds__(PA_THREADS, PA_BLOCKS) attend_k(const __grid_constant__ Attend p) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    constexpr int KEYS = PA_TILE / (HS * (int)sizeof(T)), NT = KEYS / 8;         // keys a tile, and tiles of 8
    constexpr int UNITS = HS * (int)sizeof(T) / 16;                              // 16-byte units of a row
    constexpr float SHIFT = !F32 && !BF ? 14.0f : 0.0f;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(16) AttendShared sh;
    auto &weight = sh.weight;
    auto &part_of = sh.part_of;
    auto &warp_total = sh.warp_total;
    auto &part_m = sh.part_m;
    auto &part_l = sh.part_l;
    auto &last_block = sh.last_block;
    auto *run_begin = reinterpret_cast<AttendShared::RunBegin *>(weight);
    int *group_of = reinterpret_cast<int *>(warp_total), &groups = last_block[PA_WARPS];      // first entry, last one << 8, what they say together << 16
    static_assert(sizeof(warp_total) >= 2 * PA_WARPS * sizeof(int), "");

    const Shape s = p.s;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rows_kept = min(s.group, PA_ROWS);
    unsigned char *ring = smem + w * (PA_STAGES * 2 * PA_TILE);
    // (dynamic memory: the rings, a part of a head for each warp, staged queries)
    float *first_part = reinterpret_cast<float *>(smem + PA_WARPS * PA_STAGES * 2 * PA_TILE) + w * rows_kept * HS;   // [rows][HS]
    let_successor_start();
    wait_for_predecessor();

    const int len_here = (int)blockIdx.x < s.n ? p.lens[blockIdx.x] : 1;
    if (lane < 2) part_of[w][lane] = make_int4(0, 0, 0, 0);
    Place here;
    Line line(0, 1);
    long long begin = 0;                                      // of this warp's run in the line, and its places, from 0: the next one and the end
    int at_place = 0, end = 0;
    // A warp's share of a head that a cluster has alone: to its first tile; how many there are.
    auto share_alone = [&](Place &x) {
        const int head = blockIdx.x / p.alone, warp = (blockIdx.x - head * p.alone) * PA_WARPS + w, warps = p.alone * PA_WARPS;
        x.request = head / s.vheads;
        x.vhead = head - x.request * s.vheads;
        x.len = s.length(p.lens[x.request]);
        x.tiles = s.tiles(x.len);
        x.tile = x.tiles * warp / warps;                      // (few of them)
        return x.tiles * (warp + 1) / warps - x.tile;
    };
    if (p.alone) {
        end = share_alone(here);
        __syncthreads();
    } else {
        // how many places (of one head each) lie before each thread's stretch of requests
        const int stretch = s.stretch();
        long long mine = 0;
        for (int i = 0, r = threadIdx.x * stretch; i < stretch && r < s.n; ++i, ++r) mine += s.places(p.lens[r]);
        long long sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        if (lane == 31) warp_total[w] = sum;
        __syncthreads();
        long long total = 0;
        for (int i = 0; i < PA_WARPS; ++i) {
            if (i < w) sum += warp_total[i];
            total += warp_total[i];
        }
        line = Line(total * s.vheads, gridDim.x * PA_WARPS);
        // the stretch that a run's first place lies in says so
        if (mine > 0)
#pragma unroll
            for (int i = 0; i < PA_WARPS; ++i) {
                const long long in = line.begin(blockIdx.x * PA_WARPS + i) - (sum - mine) * s.vheads;
                if (in >= 0 && in < mine * s.vheads) run_begin[i] = {in, (int)threadIdx.x * stretch};
            }
        __syncthreads();
        const int run = blockIdx.x * PA_WARPS + w;
        if (total > 0 && run < line.warps) {
            begin = line.begin(run);
            end = (int)(line.begin(run + 1) - begin);
            at_place = here.set(s, p.lens, run_begin[w].request, run_begin[w].in);
        }
    }

    if (at_place < end) {
        Place load = here;                                    // the tile that is loaded next
        int load_place = at_place;
        // queries of the first row of a head
        auto queries = [&](const Place &x) {
            return p.q + x.request * p.q_stride + (long long)((x.vhead / s.parts) * s.group + (x.vhead % s.parts) * PA_ROWS) * HS;
        };
        // ---- the ring ----
        constexpr int HELD = (KEYS + 31) / 32;
        // pages of the rows that this lane looks up, and their places in them
        struct Rows { int page[HELD], in_page[HELD]; };
        auto look_up = [&](const Place &x, Rows &rows) {
            const int *table = p.tables + (size_t)x.request * p.max_pages;
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                const unsigned key = (unsigned)x.tile * KEYS + i * 32 + lane, k = p.page_size.quotient(key);
                rows.in_page[i] = (int)(key - k * p.page_size.by);
                rows.page[i] = (KEYS >= 32 || lane < KEYS) && key < (unsigned)x.len ? table[k] : -1;
            }
        };
        unsigned valid[PA_STAGES][HELD];                      // rows that count, of each slot
        int heads_loaded = 0, heads_read = 0;                 // the staging buffer that is next (of two)
        float *staged_q = reinterpret_cast<float *>(smem + PA_WARPS * (PA_STAGES * 2 * PA_TILE + rows_kept * HS * (int)sizeof(float))) + w * 2 * rows_kept * HS;
        // (a lane's 16-byte unit is the same one of every row that it copies)
        const int lane_row = lane / UNITS, lane_unit = lane % UNITS;
        const char *lane_k = (const char *)p.c.k + lane_unit * 16, *lane_v = (const char *)p.c.v + lane_unit * 16;
        auto start_load = [&](const Rows &r, int slot) {
            long long off[HELD];                              // in bytes; 0 for a row that does not count
            unsigned rows[HELD];
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                const bool ok = (unsigned)r.page[i] < (unsigned)p.c.pages;
                off[i] = ok ? (r.page[i] * p.c.page_stride + r.in_page[i] * p.c.token_stride + (load.vhead / s.parts) * p.c.head_stride) * (long long)sizeof(T) : 0;
                rows[i] = __ballot_sync(0xffffffffu, ok);
#pragma unroll
                for (int j = 0; j < PA_STAGES; ++j)
                    if (j == slot) valid[j][i] = rows[i];
                rows[i] >>= lane_row;
            }
            unsigned char *k = ring + slot * 2 * PA_TILE, *v = k + PA_TILE;
#pragma unroll
            for (int i = 0; i < PA_TILE / 512; ++i) {
                constexpr int STEP = 32 / UNITS;              // rows an instruction
                const int row = i * STEP + lane_row, held = i * STEP / 32;
                const long long from = __shfl_sync(0xffffffffu, off[held], row & 31);
                const bool ok = rows[held] >> (i * STEP & 31) & 1;
                const int unit = F32 ? fm::unit_of(row, lane_unit) : UNITS >= 8 ? lane_unit ^ (row & 7) : lane_unit ^ ((row >> 1) & 3);
                fm::cp_async16(k + (row * UNITS + unit) * 16, lane_k + from, ok);
                fm::cp_async16(v + (row * UNITS + unit) * 16, lane_v + from, ok);
            }
            // A head's queries come with its first tile, or, where there is no room for them, on their way to L2 ahead of the reading.  Two
            // buffers: when this tile is loaded the head at hand has read its own, so only the next tile's may still have to be read.
            if (load.tile == 0) {
                const float *q = queries(load);
                const int floats = min(PA_ROWS, s.group - (load.vhead % s.parts) * PA_ROWS) * HS;
                if (p.staged) {
                    float *to = staged_q + heads_loaded * rows_kept * HS;
                    if (p.aligned_q)
                        for (int i = lane * 4; i < floats; i += 128) fm::cp_async16(to + i, q + i, true);
                    else
                        for (int i = lane; i < floats; i += 32) fm::cp_async4(to + i, q + i, true);
                    heads_loaded ^= 1;
                } else if (lane * 32 < floats) {
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(q + lane * 32));
                }
            }
            load_place += load.step();
            if (load_place < end) load.next(s, p.lens);
        };
        // ---- the head at hand ----
        // pieces of its queries: 16-bit types [HS / 16][first piece, second] (+ third for bf16), fp32 [HS / 8][4]
        uint32_t qa[F32 ? 1 : HS / 16][4], ql[BF ? HS / 16 : 1][2];
        float qf[F32 ? HS / 8 : 1][4];
        float2 o[HS / 8];
        float m = 0.0f, l = 0.0f, f = 0.0f;     // m in units of the scores as the products give them, f: log2's of one of those
        bool begins = false;
        int done = 0;                                         // parts kept for joining
        bool again = false;                                   // there are heads whose sums are not finite (NaN in their first row's output or sum says which)
        // (x: a lane's elements of q, read ahead of what else waits for memory)
        auto read_queries = [&](const float *q, float (&x)[HS / 4]) {
            const int kept = min(PA_ROWS, s.group - (here.vhead % s.parts) * PA_ROWS);
            q += g * HS;
#pragma unroll
            for (int i = 0; i < HS / 4; ++i) x[i] = g < kept ? q[16 * (i / 4) + (F32 ? 4 * t + i % 4 : 2 * t + (i & 1) + (i >> 1 & 1) * 8)] : 0.0f;
        };
        auto begin_head = [&](float (&x)[HS / 4]) {
            f = fabsf(p.scale) * 1.4426950408889634f;
            if (p.scale < 0.0f)
#pragma unroll
                for (int i = 0; i < HS / 4; ++i) x[i] = -x[i];
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < HS / 4; ++i) {
                    const float hi = round_tf32_alu(x[i]);
                    qf[i / 2][(i & 1) * 2] = hi;
                    qf[i / 2][(i & 1) * 2 + 1] = x[i] - hi;
                }
            } else {
                if (!BF) {
                    // the row's largest element to [2^14, 2^15)
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < HS / 4; ++i) top = fmaxf(top, fabsf(x[i]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int up = top > 0.0f && top < INFINITY ? min(14 - ilogbf(top), 126) : 0;
                    const float by = ldexpf(1.0f, up);
                    f = ldexpf(f, -up);
#pragma unroll
                    for (int i = 0; i < HS / 4; ++i) x[i] *= by;
                }
#pragma unroll
                for (int i = 0; i < HS / 8; ++i) {
                    uint32_t piece[BF ? 3 : 2];
                    split<T>(x[2 * i], x[2 * i + 1], piece);
                    qa[i / 2][2 * (i & 1)] = piece[0];
                    qa[i / 2][2 * (i & 1) + 1] = piece[1];
                    if (BF) ql[i / 2][i & 1] = piece[BF ? 2 : 0];
                }
            }
#pragma unroll
            for (int i = 0; i < HS / 8; ++i) o[i] = make_float2(0.0f, 0.0f);
            m = -INFINITY;
            l = 0.0f;
            begins = here.tile == 0;
        };
        // element i, e of a lane's outputs: its column
        auto column = [&](int i, int e) { return F32 ? (i / 4) * 32 + 8 * t + i % 4 + 4 * e : 8 * i + 2 * t + e; };
        auto end_head = [&](bool ends) {
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            constexpr float down = !F32 && !BF ? 1.0f / 16384.0f : 1.0f;
            const float top = m * f;                          // (-inf where nothing counted; f may be 0)
            const int kept = min(PA_ROWS, s.group - (here.vhead % s.parts) * PA_ROWS);
            l *= down;
            float2 all[4] = {make_float2(l, l == 0.0f ? 0.0f : top), o[0], o[1], o[2]};
#pragma unroll
            for (int i = 3; i < HS / 8; ++i) all[i % 4] = add2(all[i % 4], o[i]);
            all[0] = add2(add2(all[0], all[1]), add2(all[2], all[3]));
            if (__any_sync(0xffffffffu, g < kept && !(fabsf(all[0].x + all[0].y) < INFINITY))) {
                l = __int_as_float(0x7fffffff);               // NaN
                again = true;
            }
            if (begins && ends && p.alone <= 1) {
                if (g >= kept) return;
                const int h = (here.vhead / s.parts) * s.group + (here.vhead % s.parts) * PA_ROWS + g;
                float *to = p.out + here.request * p.out_stride + (long long)h * HS;
                const float by = l == 0.0f ? 0.0f : down / l;
#pragma unroll
                for (int i = 0; i < HS / 8; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) to[column(i, e)] = (e ? o[i].y : o[i].x) * by;
                if (p.lse && t == 0) p.lse[(size_t)here.request * s.heads + h] = l == 0.0f ? -INFINITY : fmaf(top, 0.6931471805599453f, logf(l));
                return;
            }
            float *to = done == 0 ? first_part : reinterpret_cast<float *>(ring);
            if (done == 1) {                                  // (the run's last head: nothing is in flight any more)
                fm::cp_wait_all();
                __syncwarp();
            }
            if (g < kept) {
#pragma unroll
                for (int i = 0; i < HS / 8; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) to[g * HS + column(i, e)] = (e ? o[i].y : o[i].x) * down;
                if (t == 0) {
                    part_m[w][done][g] = l == 0.0f ? -INFINITY : top;
                    part_l[w][done][g] = l;
                }
            }
            if (lane == 0) {
                part_of[w][done] = make_int4(here.request, here.vhead, (begins ? 1 : 0) | (ends ? 2 : 0), 1);
                if (begins && !p.alone) last_block[w] = line.warp_of(begin + at_place + here.tiles - 1 - here.tile) / PA_WARPS;
            }
            ++done;
        };

        Rows next_rows;                                       // of the tile that is loaded next
        {
            float x[HS / 4];
            read_queries(queries(here), x);
            heads_read ^= here.tile == 0;                     // (its first tile brings them again)
            Rows rows[PA_STAGES - 1];
            Place ahead = load;
            int ahead_place = load_place;
#pragma unroll
            for (int i = 0; i < PA_STAGES - 1; ++i)
                if (ahead_place < end) {
                    look_up(ahead, rows[i]);
                    ahead_place += ahead.step();
                    if (ahead_place < end) ahead.next(s, p.lens);
                }
#pragma unroll
            for (int i = 0; i < PA_STAGES - 1; ++i) {
                if (load_place < end) start_load(rows[i], i);
                fm::cp_commit();
            }
            if (load_place < end) look_up(load, next_rows);
            begin_head(x);
        }
        int slot = 0;
        while (at_place < end) {
            asm volatile("cp.async.wait_group %0;" ::"n"(PA_STAGES - 2) : "memory");
            __syncwarp();
            if (load_place < end) {
                start_load(next_rows, slot == 0 ? PA_STAGES - 1 : slot - 1);
                if (load_place < end) look_up(load, next_rows);
            }
            fm::cp_commit();
            unsigned rows[HELD];
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                rows[i] = valid[0][i];
#pragma unroll
                for (int k = 1; k < PA_STAGES; ++k)
                    if (k == slot) rows[i] = valid[k][i];
            }
            const unsigned char *kt = ring + slot * 2 * PA_TILE, *vt = kt + PA_TILE;
            const uint32_t ka = (uint32_t)__cvta_generic_to_shared(kt), va = ka + PA_TILE;
            if (++slot == PA_STAGES) slot = 0;

            // scores: keys 8 i + 2 t + e of row g
            float sc[NT][2];
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    float c[2][4] = {}, d[2][4] = {};
#pragma unroll
                    for (int jj = 0; jj < HS / 16; ++jj) {
                        const float4 x = fm::tile_ld<HS>(reinterpret_cast<const float *>(kt), 8 * i + g, 4 * jj + t);
                        const float4 h = make_float4(round_tf32_alu(x.x), round_tf32_alu(x.y), round_tf32_alu(x.z), round_tf32_alu(x.w));
                        const float2 a = add2(make_float2(x.x, x.y), make_float2(-h.x, -h.y)), b = add2(make_float2(x.z, x.w), make_float2(-h.z, -h.w));
                        mma8(c[0], qf[2 * jj], h.x, h.y);
                        mma8(c[1], qf[2 * jj + 1], h.z, h.w);
                        mma8(d[0], qf[2 * jj], a.x, a.y);
                        mma8(d[1], qf[2 * jj + 1], b.x, b.y);
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) sc[i][e] = (c[0][e] + c[1][e]) + ((c[0][2 + e] + c[1][2 + e]) + (d[0][e] + d[1][e]));
                }
            } else {
                const int id = lane >> 3;
#pragma unroll
                for (int i = 0; i < NT; i += 2) {
                    float c[2][2][4] = {}, d[2][4] = {};
                    const int row = 8 * i + (lane & 7) + (id >> 1) * 8;
#pragma unroll
                    for (int jj = 0; jj < HS / 16; ++jj) {
                        const int u = 2 * jj + (id & 1);
                        uint32_t b[4];
                        ldmatrix4<false>(b, ka + (row * UNITS + (UNITS >= 8 ? u ^ (row & 7) : u ^ ((row >> 1) & 3))) * 16);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            mma16(c[k][jj & 1], qa[jj][0], qa[jj][1], qa[jj][2], qa[jj][3], b[2 * k], b[2 * k + 1], T());
                            if constexpr (BF) mma16(d[k], ql[jj][0], 0, ql[jj][1], 0, b[2 * k], b[2 * k + 1], T());
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float2 x = add2(add2(make_float2(c[k][0][0], c[k][0][1]), make_float2(c[k][1][0], c[k][1][1])),
                                              add2(add2(make_float2(c[k][0][2], c[k][0][3]), make_float2(c[k][1][2], c[k][1][3])), make_float2(d[k][0], d[k][1])));
                        sc[i + k][0] = x.x;
                        sc[i + k][1] = x.y;
                    }
                }
            }
            // weights
            bool full = true;                                 // all rows count
#pragma unroll
            for (int i = 0; i < HELD; ++i) full = full && rows[i] == (KEYS >= 32 ? ~0u : (1u << (KEYS & 31)) - 1);
            if (!full)
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (!(rows[i / 4] >> (8 * (i % 4) + 2 * t + e) & 1)) sc[i][e] = -INFINITY;
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < NT; ++i) top = fmaxf(top, fmaxf(sc[i][0], sc[i][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (__any_sync(0xffffffffu, top > m)) {
                const float mn = fmaxf(m, top), by = m == -INFINITY ? 0.0f : two_to((m - mn) * f);
                l *= by;
#pragma unroll
                for (int i = 0; i < HS / 8; ++i) { o[i].x *= by; o[i].y *= by; }
                m = mn;
            }
            const float from = m == -INFINITY ? 0.0f : m;
            // (the weight of a row that does not count is 0 also where f is 0)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = two_to(fmaf(sc[i][e] - from, f, SHIFT));
                    sc[i][e] = full || (rows[i / 4] >> (8 * (i % 4) + 2 * t + e) & 1) ? x : 0.0f;
                    l += sc[i][e];
                }
            // weights times values
            if constexpr (F32) {
                float pw[NT][4];
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        pw[i][2 * e] = round_tf32_alu(sc[i][e]);
                        pw[i][2 * e + 1] = sc[i][e] - pw[i][2 * e];
                    }
#pragma unroll
                for (int d = 0; d < HS / 32; ++d) {
                    float c[4][4] = {};
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        const float4 x = fm::tile_ld<HS>(reinterpret_cast<const float *>(vt), 8 * i + 2 * t, 8 * d + g);
                        const float4 y = fm::tile_ld<HS>(reinterpret_cast<const float *>(vt), 8 * i + 2 * t + 1, 8 * d + g);
                        const float a[4] = {x.x, x.y, x.z, x.w}, b[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float ah = round_tf32_alu(a[e]), bh = round_tf32_alu(b[e]);
                            const float2 r = add2(make_float2(a[e], b[e]), make_float2(-ah, -bh));
                            mma8(c[e], pw[i], ah, bh);
                            mma8(c[e], pw[i], r.x, r.y);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[4 * d + e] = add2(o[4 * d + e], add2(make_float2(c[e][0], c[e][1]), make_float2(c[e][2], c[e][3])));
                }
            } else {
                uint32_t pw[NT][BF ? 3 : 2];
#pragma unroll
                for (int i = 0; i < NT; ++i) split<T>(sc[i][0], sc[i][1], pw[i]);
                const int id = lane >> 3;
#pragma unroll
                for (int d = 0; d < HS / 16; ++d) {
                    float c[2][4] = {};
#pragma unroll
                    for (int i = 0; i < NT; i += 2) {
                        const int row = 8 * i + (lane & 7) + (id & 1) * 8, u = 2 * d + (id >> 1);
                        uint32_t b[4];
                        ldmatrix4<true>(b, va + (row * UNITS + (UNITS >= 8 ? u ^ (row & 7) : u ^ ((row >> 1) & 3))) * 16);
                        mma16(c[0], pw[i][0], pw[i][1], pw[i + 1][0], pw[i + 1][1], b[0], b[1], T());
                        mma16(c[1], pw[i][0], pw[i][1], pw[i + 1][0], pw[i + 1][1], b[2], b[3], T());
                        if constexpr (BF) {
                            mma16(c[0], pw[i][2], 0, pw[i + 1][2], 0, b[0], b[1], T());
                            mma16(c[1], pw[i][2], 0, pw[i + 1][2], 0, b[2], b[3], T());
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) o[2 * d + k] = add2(o[2 * d + k], add2(make_float2(c[k][0], c[k][1]), make_float2(c[k][2], c[k][3])));
                }
            }
            const bool ends = here.tile + 1 == here.tiles, last = at_place + here.step() >= end;
            if (ends || last) end_head(ends);
            at_place += here.step();
            if (!last) here.next(s, p.lens);
            if (ends && !last) {
                // the queries staged with the tile that is next, which has to have come
                if (p.staged) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(PA_STAGES - 2) : "memory");
                    __syncwarp();
                }
                float x[HS / 4];
                read_queries(p.staged ? staged_q + heads_read * rows_kept * HS : queries(here), x);
                heads_read ^= 1;
                begin_head(x);
            }
        }

        // ---- heads whose sums are not finite, once more and without pieces ----
        if (again) {
            __syncwarp();
            Place x;
            int at = 0, part = 0;
            if (p.alone) share_alone(x);
            else at = x.set(s, p.lens, run_begin[w].request, run_begin[w].in);
            while (at < end) {
                const int t0 = x.tile, t1 = min(x.tiles, t0 + (end - at));
                const bool whole = t0 == 0 && t1 == x.tiles && p.alone <= 1;
                const int kept = min(PA_ROWS, s.group - (x.vhead % s.parts) * PA_ROWS), h0 = (x.vhead / s.parts) * s.group + (x.vhead % s.parts) * PA_ROWS;
                float *to = whole ? p.out + x.request * p.out_stride + (long long)h0 * HS : part == 0 ? first_part : reinterpret_cast<float *>(ring);
                const float found = whole ? to[0] : part_l[w][part][0];
                if (found != found) {
                    const int *table = p.tables + (size_t)x.request * p.max_pages;
                    const int first = t0 * KEYS, behind = (int)min((long long)t1 * KEYS, (long long)x.len);
                    for (int r = 0; r < kept; ++r) {
                        float xq[HS / 32], y[HS / 32] = {}, top = -INFINITY, sum = 0.0f;      // columns lane, lane + 32, ...
#pragma unroll
                        for (int i = 0; i < HS / 32; ++i) xq[i] = queries(x)[r * HS + lane + 32 * i];
#pragma unroll 1
                        for (int key = first; key < behind; ++key) {
                            const unsigned k = p.page_size.quotient(key);
                            const int page = table[k];
                            if ((unsigned)page >= (unsigned)p.c.pages) continue;
                            const long long off = page * p.c.page_stride + (int)(key - k * p.page_size.by) * p.c.token_stride + (x.vhead / s.parts) * p.c.head_stride + lane;
                            float score = 0.0f;
#pragma unroll
                            for (int i = 0; i < HS / 32; ++i) score = fmaf(xq[i], (float)((const T *)p.c.k)[off + 32 * i], score);
                            score = warp_sum(score) * p.scale * 1.4426950408889634f;
                            const float mn = fmaxf(top, score), by = top == -INFINITY ? 0.0f : exp2f(top - mn);
                            const float weigh = score == -INFINITY ? 0.0f : exp2f(score - mn);
                            sum = fmaf(sum, by, weigh);
#pragma unroll
                            for (int i = 0; i < HS / 32; ++i) y[i] = fmaf(weigh, (float)((const T *)p.c.v)[off + 32 * i], y[i] * by);
                            top = mn;
                        }
                        const float over = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                        for (int i = 0; i < HS / 32; ++i) to[r * HS + lane + 32 * i] = y[i] * over;
                        if (lane == 0) {
                            if (!whole) {
                                part_m[w][part][r] = sum == 0.0f ? -INFINITY : top;
                                part_l[w][part][r] = sum;
                            } else if (p.lse) {
                                p.lse[(size_t)x.request * s.heads + h0 + r] = sum == 0.0f ? -INFINITY : fmaf(top, 0.6931471805599453f, logf(sum));
                            }
                        }
                    }
                }
                part += !whole;
                at += t1 - t0 + 1;
                if (at < end) {
                    x.tile = x.tiles - 1;
                    x.next(s, p.lens);
                }
            }
        }
    }

    // ---- heads that several of the block's warps, or blocks, have parts of ----
    __syncthreads();
    // A group is a head's entries one behind the other.  Each entry's weight in its group, a thread for each row; and the groups.
    static_assert(2 * PA_WARPS * PA_ROWS <= PA_THREADS && 2 * PA_WARPS <= 32, "");
    auto entry = [&](int i) { return part_of[i >> 1][i & 1]; };
    auto same = [](int4 a, int4 b) { return a.w && b.w && a.x == b.x && a.y == b.y; };
    if (threadIdx.x < 2 * PA_WARPS * PA_ROWS) {
        const int e = threadIdx.x / PA_ROWS, r = threadIdx.x % PA_ROWS;
        const int4 of = entry(e);
        float top = LOWEST;                                   // (so that the weight of a maximum of -infinity is 0)
#pragma unroll
        for (int i = 0; i < 2 * PA_WARPS; ++i)
            if (same(of, entry(i))) top = fmaxf(top, part_m[i >> 1][i & 1][r]);
        weight[e][r] = of.w ? exp2f(part_m[e >> 1][e & 1][r] - top) : -1.0f;      // (below 0: there is none)
    } else if (w == PA_WARPS - 1) {
        const int4 of = lane < 2 * PA_WARPS ? entry(lane) : make_int4(0, 0, 0, 0);
        bool first = of.w;
        int last = lane, flags = of.z;
#pragma unroll
        for (int i = 0; i < 2 * PA_WARPS; ++i)
            if (same(of, entry(i))) {
                if (i < lane) first = false;
                if (i > lane) last = i;
                flags |= entry(i).z;
            }
        const unsigned firsts = __ballot_sync(0xffffffffu, first);
        if (first) group_of[__popc(firsts & ((1u << lane) - 1))] = lane | last << 8 | flags << 16;
        if (first && flags == 1 && !p.alone) p.w.begun[blockIdx.x] = make_int4(of.x, of.y, last_block[lane >> 1], 1);
        if (lane == 0) groups = __popc(firsts);
        if (!__any_sync(0xffffffffu, first && flags == 1) && lane == 0 && !p.alone) p.w.begun[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
    // (of a cluster: the block's part of the head, in the second place of the first warp's ring)
    float *block_o = reinterpret_cast<float *>(smem + 2 * PA_TILE), *block_m = block_o + PA_ROWS * HS, *block_l = block_m + PA_ROWS;
    static_assert(PA_ROWS * (HS + 2) * sizeof(float) <= 2 * PA_TILE, "");
    if (p.alone > 1 && threadIdx.x < PA_ROWS) {               // (none, if it has no tile)
        block_m[threadIdx.x] = -INFINITY;
        block_l[threadIdx.x] = -1.0f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < groups * rows_kept * (HS / 4); i += PA_THREADS) {
        const int row_in = i / (HS / 4), d = i % (HS / 4) * 4, r = row_in % rows_kept;
        const int gr = group_of[row_in / rows_kept], e0 = gr & 255, e1 = gr >> 8 & 255, flags = gr >> 16;
        const int4 of = entry(e0);
        const int h = (of.y / s.parts) * s.group + (of.y % s.parts) * PA_ROWS + r;
        if (r >= s.group - (of.y % s.parts) * PA_ROWS) continue;
        float all = 0.0f, top = -INFINITY, x[4] = {};
#pragma unroll
        for (int k = 0; k < 2 * PA_WARPS; ++k) {
            const float by = k < e0 || k > e1 ? -1.0f : weight[k][r];     // (below 0 also for an entry between them that is none)
            const float4 v = *reinterpret_cast<const float4 *>(
                (k & 1 ? smem + (k >> 1) * (PA_STAGES * 2 * PA_TILE) : smem + PA_WARPS * PA_STAGES * 2 * PA_TILE + (k >> 1) * rows_kept * HS * sizeof(float)) +
                (r * HS + d) * sizeof(float));
            const bool use = !(by < 0.0f);                    // (a weight of 0 is one: 0 times an infinity or NaN is NaN)
            all = use ? fmaf(part_l[k >> 1][k & 1][r], by, all) : all;
            top = use ? fmaxf(top, part_m[k >> 1][k & 1][r]) : top;
            x[0] = use ? fmaf(v.x, by, x[0]) : x[0];
            x[1] = use ? fmaf(v.y, by, x[1]) : x[1];
            x[2] = use ? fmaf(v.z, by, x[2]) : x[2];
            x[3] = use ? fmaf(v.w, by, x[3]) : x[3];
        }
        if (p.alone > 1) {
            *reinterpret_cast<float4 *>(block_o + r * HS + d) = make_float4(x[0], x[1], x[2], x[3]);
            if (d == 0) {
                block_m[r] = top;
                block_l[r] = all;
            }
        } else if (flags == 3) {
            float *to = p.out + of.x * p.out_stride + (long long)h * HS + d;
            const float by = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
            for (int j = 0; j < 4; ++j) to[j] = x[j] * by;
            if (p.lse && d == 0) p.lse[(size_t)of.x * s.heads + h] = all == 0.0f ? -INFINITY : fmaf(top, 0.6931471805599453f, logf(all));
        } else {
            const size_t row = ((size_t)blockIdx.x * 2 + (flags & 1)) * PA_ROWS + r;
            *reinterpret_cast<float4 *>(p.w.o + row * HS + d) = make_float4(x[0], x[1], x[2], x[3]);
            if (d == 0) {
                p.w.m[row] = top;
                p.w.l[row] = all;
            }
        }
    }
    if (p.alone > 1) {
        // the cluster's blocks join their parts, a share of the elements each
        cluster_sync();
        const int head = blockIdx.x / p.alone, request = head / s.vheads, vhead = head - request * s.vheads;
        const int kept = min(PA_ROWS, s.group - (vhead % s.parts) * PA_ROWS), h0 = (vhead / s.parts) * s.group + (vhead % s.parts) * PA_ROWS;
        for (int i = (blockIdx.x - head * p.alone) * PA_THREADS + threadIdx.x; i < kept * (HS / 4); i += p.alone * PA_THREADS) {
            const int r = i / (HS / 4), d = i % (HS / 4) * 4;
            float m[PA_CLUSTER], l[PA_CLUSTER], top = LOWEST, all = 0.0f, x[4] = {};
            float4 v[PA_CLUSTER];
#pragma unroll
            for (int k = 0; k < PA_CLUSTER; ++k) {
                m[k] = -INFINITY;
                l[k] = -1.0f;
                if (k >= p.alone) continue;
                m[k] = read_of<float>(block_m + r, k);
                l[k] = read_of<float>(block_l + r, k);
                v[k] = read_of<float4>(block_o + r * HS + d, k);
                top = fmaxf(top, m[k]);
            }
#pragma unroll
            for (int k = 0; k < PA_CLUSTER; ++k) {
                if (l[k] < 0.0f) continue;
                const float by = exp2f(m[k] - top);
                all = fmaf(l[k], by, all);
                x[0] = fmaf(v[k].x, by, x[0]);
                x[1] = fmaf(v[k].y, by, x[1]);
                x[2] = fmaf(v[k].z, by, x[2]);
                x[3] = fmaf(v[k].w, by, x[3]);
            }
            float *to = p.out + request * p.out_stride + (long long)(h0 + r) * HS + d;
            const float by = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
            for (int j = 0; j < 4; ++j) to[j] = x[j] * by;
            if (p.lse && d == 0) p.lse[(size_t)request * s.heads + h0 + r] = all == 0.0f ? -INFINITY : fmaf(top, 0.6931471805599453f, logf(all));
        }
        cluster_sync();                                       // (the others have read this block's part)
    }
    // ---- requests without tokens ----  (a row, and what is behind the last request or head, may be beyond an int)
    for (long long r = blockIdx.x; r < s.n; r += gridDim.x) {
        if (s.length(r == blockIdx.x ? len_here : p.lens[r]) > 0) continue;
        for (long long i = threadIdx.x; i < (long long)s.heads * HS; i += PA_THREADS) p.out[r * p.out_stride + i] = 0.0f;
        if (p.lse)
            for (long long h = threadIdx.x; h < s.heads; h += PA_THREADS) p.lse[r * s.heads + h] = -INFINITY;
    }
}

// The heads that reach over blocks: a block for each block of attend_k that began one, and each row.  Parts are read 16 to 64 at a
// time and four of those ahead of the sums: with two at a time one head in 132 parts took 8 us.
constexpr int PJ_THREADS = 512;
template <int HS>
__global__ void __launch_bounds__(PJ_THREADS) attend_join_k(const __grid_constant__ Attend p) {
    constexpr int ACROSS = PJ_THREADS * 4 / HS, HELD = PA_MOST_BLOCKS / PJ_THREADS;
    __shared__ float by[PA_MOST_BLOCKS], red[32], sum[ACROSS][HS];
    const Shape s = p.s;
    const int r = blockIdx.y, d = threadIdx.x % (HS / 4) * 4, a = threadIdx.x / (HS / 4);
    let_successor_start();
    wait_for_predecessor();
    const int4 of = p.w.begun[blockIdx.x];
    if (!of.w || r >= min(PA_ROWS, s.group - (of.y % s.parts) * PA_ROWS)) return;
    const int b0 = blockIdx.x, n = of.z - b0 + 1;             // parts: the second of block b0, the first of those behind it
    auto row = [&](int i) { return ((size_t)(b0 + i) * 2 + (i == 0 ? 1 : 0)) * PA_ROWS + r; };
    float m[HELD], l[HELD], top = -INFINITY, all = 0.0f;
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int i = threadIdx.x + k * PJ_THREADS;
        m[k] = i < n ? p.w.m[row(i)] : -INFINITY;
        l[k] = i < n ? p.w.l[row(i)] : 0.0f;
        top = fmaxf(top, m[k]);
    }
    constexpr int AHEAD = 4;
    float4 v[AHEAD];
    auto read = [&](int i) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            v[k] = i + k * ACROSS < n ? *reinterpret_cast<const float4 *>(p.w.o + row(i + k * ACROSS) * HS + d) : make_float4(0, 0, 0, 0);
    };
    read(a);
    // (a maximum of -inf, which block_reduce raises to the lowest number, has no weights: l is 0 throughout, or NaN)
    top = block_reduce<true>(top, red);
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const float x = l[k] == 0.0f ? 0.0f : exp2f(m[k] - top);
        if (threadIdx.x + k * PJ_THREADS < n) by[threadIdx.x + k * PJ_THREADS] = x;
        all += l[k] * x;
    }
    all = block_reduce<false>(all, red);                      // (its barriers also publish the weights)
    float x[4] = {};
    for (int i = a; i < n; i += AHEAD * ACROSS) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const float w = i + k * ACROSS < n ? by[i + k * ACROSS] : 0.0f;
            x[0] = fmaf(v[k].x, w, x[0]);
            x[1] = fmaf(v[k].y, w, x[1]);
            x[2] = fmaf(v[k].z, w, x[2]);
            x[3] = fmaf(v[k].w, w, x[3]);
        }
        read(i + AHEAD * ACROSS);
    }
    *reinterpret_cast<float4 *>(&sum[a][d]) = make_float4(x[0], x[1], x[2], x[3]);
    __syncthreads();
    if (threadIdx.x < HS) {
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < ACROSS; ++i) y += sum[i][threadIdx.x];
        const int h = (of.y / s.parts) * s.group + (of.y % s.parts) * PA_ROWS + r;
        p.out[of.x * p.out_stride + (long long)h * HS + threadIdx.x] = all == 0.0f ? 0.0f : y / all;
        if (p.lse && threadIdx.x == 0) p.lse[(size_t)of.x * s.heads + h] = all == 0.0f ? -INFINITY : fmaf(top, 0.6931471805599453f, logf(all));
    }
}

size_t element(int type) { return type == BMB_TYPE_FP32 ? 4 : 2; }

int check_cache(const char *what, const bmb_kv_cache *c) {
    if (!c || !c->k || !c->v) return fail(BMB_E_ARG, "%s: no cache", what);
    if (c->type < BMB_TYPE_FP32 || c->type > BMB_TYPE_FP16) return fail(BMB_E_ARG, "%s: unknown type %d", what, c->type);
    if (c->pages <= 0 || c->page_size <= 0 || c->heads <= 0)
        return fail(BMB_E_ARG, "%s: bad sizes (pages=%d page_size=%d heads=%d)", what, c->pages, c->page_size, c->heads);
    if (c->head_size != 32 && c->head_size != 64 && c->head_size != 128)
        return fail(BMB_E_UNSUPPORTED, "%s: head size %d (32, 64 and 128 are served)", what, c->head_size);
    if ((long long)c->heads * c->head_size > INT_MAX) return fail(BMB_E_LIMIT, "%s: %d heads", what, c->heads);
    if ((long long)c->pages * c->page_size > INT_MAX) return fail(BMB_E_LIMIT, "%s: %d pages of %d tokens are beyond an int", what, c->pages, c->page_size);
    const long long unit = 16 / (long long)element(c->type);
    const long long strides[] = {c->page_stride, c->token_stride, c->head_stride};
    for (long long s : strides)
        if (s < c->head_size || s % unit) return fail(BMB_E_ARG, "%s: stride %lld (multiples of 16 bytes, at least the head size)", what, s);
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return fail(BMB_E_ARG, "%s: the cache is not 16-byte aligned", what);
    return BMB_OK;
}

Shape attend_shape(int n, int heads, int kv_heads, int hs, int type, int cap) {
    Shape s;
    s.n = n;
    s.heads = heads;
    s.group = heads / kv_heads;
    s.parts = ceil_div(s.group, PA_ROWS);
    s.vheads = kv_heads * s.parts;
    s.cap = cap;
    s.keys_log2 = 0;
    while ((PA_TILE >> s.keys_log2) > hs * (int)element(type)) ++s.keys_log2;
    return s;
}

template <typename T, int HS>
int run_attend(Attend &p, cudaStream_t st) {
    const int blocks = attend_blocks(), rows = p.s.group < PA_ROWS ? p.s.group : PA_ROWS;
    // staged queries where two blocks still fit an SM
    const size_t part = rows * HS * sizeof(float), least = (size_t)PA_WARPS * (PA_STAGES * 2 * PA_TILE + part);
    p.staged = least + PA_WARPS * 2 * part <= PA_SMEM;
    p.aligned_q = ((uintptr_t)p.q & 15) == 0 && p.q_stride % 4 == 0;
    static std::atomic<unsigned long long> prepared{0};       // devices (those from 64 on are prepared every time)
    const int dev = current_device();
    const unsigned long long bit = dev >= 0 && dev < 64 ? 1ULL << dev : 0;
    if (!(prepared.load(std::memory_order_relaxed) & bit)) {
        BMB_CUDA(cudaFuncSetAttribute(attend_k<T, HS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PA_SMEM));
        prepared.fetch_or(bit, std::memory_order_relaxed);
    }
    const size_t smem = least + (p.staged ? PA_WARPS * 2 * part : 0);
    if (p.alone) return launch_cluster(attend_k<T, HS>, p.s.n * p.s.vheads * p.alone, p.alone, PA_THREADS, smem, st, p);
    BMB_TRY(launch_in_chain(attend_k<T, HS>, blocks, PA_THREADS, smem, st, p));
    return launch_in_chain(attend_join_k<HS>, dim3(blocks, rows), PJ_THREADS, 0, st, p);
}
template <typename T>
int run_attend(Attend &p, cudaStream_t st) {
    switch (p.c.head_size) {
    case 32: return run_attend<T, 32>(p, st);
    case 64: return run_attend<T, 64>(p, st);
    default: return run_attend<T, 128>(p, st);
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
    if (!k || !v || !slots || !words(k, v, slots)) return fail(BMB_E_ARG, "paged_kv_write: a null or unaligned pointer");
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->type == BMB_TYPE_FP32) return run_write<float>(*cache, k, v, row_stride, slots, tokens, st);
    if (cache->type == BMB_TYPE_BF16) return run_write<__nv_bfloat16>(*cache, k, v, row_stride, slots, tokens, st);
    return run_write<__half>(*cache, k, v, row_stride, slots, tokens, st);
}

size_t bmb_paged_attention_workspace(int heads, int kv_heads, int head_size) {
    (void)heads;
    (void)kv_heads;
    return attend_workspace(attend_blocks(), head_size);
}

int bmb_paged_attention_schedule_check(const int *host_lens, int n, int heads, int kv_heads, int head_size, int type, int max_len, int blocks,
                                       long long *tiles_out, int *joined_out) {
    if (!host_lens || n <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_len <= 0 || blocks <= 0 || blocks > PA_MOST_BLOCKS || type < BMB_TYPE_FP32 || type > BMB_TYPE_FP16 ||
        (head_size != 32 && head_size != 64 && head_size != 128))
        return fail(BMB_E_ARG, "paged_attention_schedule_check: bad argument");
    const Shape s = attend_shape(n, heads, kv_heads, head_size, type, max_len);
    long long total = 0, tiles = 0, done = 0;
    std::vector<long long> before;                            // as a block counts them
    for (int r = 0; r < n; ++r) {
        if (r % s.stretch() == 0) before.push_back(total);
        total += s.places(host_lens[r]);
        tiles += (long long)s.tiles(host_lens[r]) * s.vheads;
    }
    const Line line(total * s.vheads, blocks * PA_WARPS);
    int joined = 0;
    std::vector<int> goes_on(blocks, 0);                      // blocks that have a part of the head that an earlier block began
    std::vector<int> promised(blocks, 0);
    Place all{-1, s.vheads - 1, 0, 0, 0};                     // the line from its first tile to its last
    for (int w = 0; total > 0 && w < line.warps; ++w) {
        int at = 0, parts = 0;
        while (at < (int)before.size() && before[at] * s.vheads <= line.begin(w)) ++at;
        Place here;
        const long long begin = line.begin(w), end = line.begin(w + 1);
        long long place = begin + here.set(s, host_lens, (at - 1) * s.stretch(), begin - before[at - 1] * s.vheads);
        bool begins = here.tile == 0;
        while (place < end) {
            all.next(s, host_lens);
            ++done;
            if (here.request >= n || here.request != all.request || here.vhead != all.vhead || here.tile != all.tile || line.warp_of(place) != w)
                return fail(BMB_E_ARG, "paged_attention_schedule_check: warp %d has another tile at %lld", w, place);
            const bool ends = here.tile + 1 == here.tiles, last = place + here.step() >= end;
            if (ends || last) {
                if (!(begins && ends) && ++parts > 2) return fail(BMB_E_ARG, "paged_attention_schedule_check: warp %d has %d parts", w, parts);
                const int b = w / PA_WARPS, first_block = line.warp_of(place - here.tile) / PA_WARPS;
                const int last_block = line.warp_of(place + here.tiles - 1 - here.tile) / PA_WARPS;
                if (first_block < b) goes_on[b] = first_block + 1;
                if (first_block == b && last_block > b) {
                    if (promised[b] != last_block) ++joined;
                    promised[b] = last_block;
                }
                begins = true;
            }
            place += here.step();
            here.next(s, host_lens);
        }
    }
    if (done != tiles) return fail(BMB_E_ARG, "paged_attention_schedule_check: %lld of %lld tiles", done, tiles);
    for (int b = 0; b < blocks; ++b)
        for (int i = b + 1; i <= promised[b]; ++i)
            if (goes_on[i] != b + 1) return fail(BMB_E_ARG, "paged_attention_schedule_check: block %d has no part of block %d's head", i, b);
    if (tiles_out) *tiles_out = tiles;
    if (joined_out) *joined_out = joined;
    return BMB_OK;
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
    if (!out || !q || !tables || !lens || !words(out, lse, q, tables, lens)) return fail(BMB_E_ARG, "paged_attention: a null or unaligned pointer");
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < bmb_paged_attention_workspace(heads, cache->heads, cache->head_size))
        return fail(BMB_E_ARG, "paged_attention: a workspace of %zu bytes, 16-byte aligned, is needed (got %zu)",
                    bmb_paged_attention_workspace(heads, cache->heads, cache->head_size), workspace_bytes);
    Attend p{};
    p.out = out;
    p.lse = lse;
    p.q = q;
    p.c = *cache;
    p.tables = tables;
    p.lens = lens;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.max_pages = max_pages;
    p.page_size = Divide((unsigned)cache->page_size);
    p.scale = scale;
    const int hs = cache->head_size, blocks = attend_blocks();
    p.s = attend_shape(n, heads, cache->heads, hs, cache->type, max_pages * cache->page_size);
    if ((double)n * p.s.vheads * p.s.places(p.s.cap) > 1e12)
        return fail(BMB_E_LIMIT, "paged_attention: %d requests of %d tokens", n, p.s.cap);
    p.alone = blocks_alone((long long)n * p.s.vheads, p.s.tiles(p.s.cap), blocks);
    p.w.o = (float *)workspace;
    p.w.m = p.w.o + (size_t)blocks * 2 * PA_ROWS * hs;
    p.w.l = p.w.m + (size_t)blocks * 2 * PA_ROWS;
    p.w.begun = (int4 *)((char *)workspace + attend_workspace(blocks, hs) - (size_t)blocks * sizeof(int4));
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->type == BMB_TYPE_FP32) return run_attend<float>(p, st);
    if (cache->type == BMB_TYPE_BF16) return run_attend<__nv_bfloat16>(p, st);
    return run_attend<__half>(p, st);
}

}  // extern "C"
