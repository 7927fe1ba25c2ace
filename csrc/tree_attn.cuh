// Shared pieces of the tensor-core tree attention kernels (tree_attn_sm100.cu: tiles of 16 query rows on mma.sync,
// tree_attn_tile_sm100.cu: tiles of 128 rows on tcgen05): parameters, the cut of the work, the merge of partial results.
#pragma once
#include <cuda_fp8.h>

#include "tc.cuh"

typedef __nv_bfloat16 bf16;

namespace tree {

constexpr int PAGE = 16, MAX_B = 1024;
// 8-bit pages: most binary orders of magnitude between the powers of two of a unit's values for one unit of the output, in which 16-bit operands
// carry them: a row's terms are then off by at most 2^-17 of its largest, whatever tokens it does not see or gives no weight (2^-25 where it sees the
// largest values).  Values further apart (hidden ones count: what they hold is not known to be small) are added in fp32 where rows are few,
// or have a unit per row that follows the row's own terms.  (Normal numbers times lognormal factors of e^0.7 lie within 2^9 in a part of a thousand
// tokens.  The rare path takes 7 and 2.5 times as long.)
constexpr int SPREAD = 12;
constexpr float NO_UNIT = -1e30f;                      // log2 of the unit of an output without a term

struct TreeParams {
    const bf16* q;
    long long q_stride;
    const uint8_t *k, *v, *ke, *ve;                    // pages, and exponents of 8-bit pages
    const int *table, *ctx_lens, *cu;
    const long long* masks;
    bf16* out;
    long long out_stride;
    float* part_o;                                     // [2 * workers][ROWS][HD], or [2 * workers][HD / 4][ROWS][4] (128 rows)
    float* part_ml;                                    // [2 * workers][ROWS][2]
    int* uoff;                                         // [B + 1] tiles before each sequence, for the merge kernel
    int max_pages, num_pages, B, N, H, G, n_kv, max_q, max_ctx;
    float scale_log2;
    int* status;
    int row_blocks, zero_tail;                         // a block of threads per unit: blocks of rows that a sequence may have; rows that are no sequence's -> 0
};

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) { return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ uint32_t largest(uint32_t two_bf16) { return max(two_bf16 & 0x7fffu, (two_bf16 >> 16) & 0x7fffu); }
// Four bf16 numbers times `inv` as the sum of two e4m3 numbers each: together they hold the eight bits of a bf16 number from 2^-2 on; smaller
// ones are off by at most 2^-10.
__device__ __forceinline__ void split_e4m3(uint2 q, float inv, uint32_t& hi, uint32_t& lo) {
    uint32_t h[2], l[2];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        const uint32_t w = z ? q.y : q.x;
        const float a = __uint_as_float(w << 16) * inv, b = __uint_as_float(w & 0xffff0000u) * inv;
        h[z] = e4m3x2(a, b);
        const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)h[z], __NV_E4M3)));
        l[z] = e4m3x2(a - back.x, b - back.y);
    }
    hi = h[0] | h[1] << 16;
    lo = l[0] | l[1] << 16;
}
// Least biased exponent of the power of two that is taken out of a query row (rows of zeros and of numbers below 2^-119 have this one): its
// place below is then a normal number, which arithmetic that takes denormal numbers for zero keeps, and no hidden score (-infinity) meets a zero.
constexpr int Q_LEAST = 8;
// The power of two that brings a row's largest number to [2^7, 2^8), from the largest magnitude's bits, and its inverse; NaN where the row is not finite.
__device__ __forceinline__ float q_down(uint32_t big) {
    return big >= 0x7f80u ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(261 - max((int)(big >> 7), Q_LEAST)) << 23);
}
__device__ __forceinline__ float q_up(uint32_t big) { return __uint_as_float((uint32_t)(max((int)(big >> 7), Q_LEAST) - 7) << 23); }
// four e4m3 codes -> two f16 pairs
__device__ __forceinline__ void codes_to_f16(uint32_t c, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(c));
}
__device__ __forceinline__ float pow2_biased(int b) { return __uint_as_float(b > 0 ? (uint32_t)b << 23 : 0x00400000u); }
// Pages are fetched 16 bytes per thread.  (A TMA copy costs ~150 cycles of its engine whatever its size: blocks of 2 KB, a page of one
// head, reached 3.4 TB/s over the GPU, 16-byte copies by the threads 6.8.)
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Arrives on `bar` when this thread's copies so far have landed (counted among the barrier's arrivals).
__device__ __forceinline__ void copy_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// rows of a sequence and its tokens; 0 rows where it has none or breaks the rules
__device__ __forceinline__ int2 span_of(const TreeParams& p, int b, bool report) {
    const int c0 = p.cu ? p.cu[b] : b, c1 = p.cu ? p.cu[b + 1] : b + 1, n = c1 - c0, ctx = p.ctx_lens[b];
    if (n <= 0) return make_int2(0, 0);
    if (c0 < 0 || c1 > p.N || n > p.max_q || n > 64 || n > ctx || ctx > p.max_ctx || (ctx + PAGE - 1) / PAGE > p.max_pages) {
        if (report && p.status) atomicMax(p.status, (int)KB_BAD_INDEX);
        return make_int2(0, 0);
    }
    return make_int2(n, ctx);
}

struct Segment {                                       // a worker's part of one unit
    int b, h, rb, n, ctx, T, t0, t1;
};
// The unit of tile x, as far as a part that ends at `hi` has it from x on.
template <int ROWS, int TILE>
__device__ __forceinline__ Segment segment_at(const TreeParams& p, const int* uoff, int x, int hi) {
    int a = 0, z = p.B;
    while (z - a > 1) {
        const int m = (a + z) >> 1;
        if (uoff[m] <= x) a = m; else z = m;
    }
    Segment s;
    s.b = a;
    const int2 sp = span_of(p, a, false);
    s.n = sp.x;
    s.ctx = sp.y;
    s.T = (sp.y + TILE - 1) / TILE;
    const int rel = x - uoff[a], unit = rel / s.T, rbs = (sp.x * p.G + ROWS - 1) / ROWS;
    s.h = unit / rbs;
    s.rb = unit % rbs;
    s.t0 = rel - unit * s.T;
    s.t1 = min(s.T, s.t0 + hi - x);
    return s;
}
// Tiles before each sequence -> uoff[0 .. B] (shared memory), by all threads of the block; block 0 leaves them for the merge kernel.
template <int ROWS, int TILE, int THREADS>
__device__ __forceinline__ void count_tiles(const TreeParams& p, int* uoff, int* wsum) {
    const int per = (p.B + THREADS - 1) / THREADS, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int mine = 0;
    for (int i = 0; i < per; ++i) {
        const int b = threadIdx.x * per + i;
        if (b >= p.B) break;
        const int2 s = span_of(p, b, blockIdx.x == 0);
        const int t = p.n_kv * ((s.x * p.G + ROWS - 1) / ROWS) * ((s.y + TILE - 1) / TILE);
        uoff[b + 1] = t;
        mine += t;
    }
    int s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += v;
    }
    if (lane == 31) wsum[warp] = s;
    __syncthreads();
    int run = s - mine;
    for (int w = 0; w < warp; ++w) run += wsum[w];
    for (int i = 0; i < per; ++i) {
        const int b = threadIdx.x * per + i;
        if (b >= p.B) break;
        run += uoff[b + 1];
        uoff[b + 1] = run;
    }
    if (threadIdx.x == 0) uoff[0] = 0;
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i <= p.B; i += THREADS) p.uoff[i] = uoff[i];
}
// The part [lo, hi) of the line of tiles that worker `w` of `workers` has (empty where there are more workers than tiles: every part that
// exists has a tile, since the merge reads all parts between a unit's first and last).
__device__ __forceinline__ int2 part_of_line(long long total, int w, int workers) {
    const long long parts = min((long long)workers, total);
    if (w >= parts) return make_int2(0, 0);
    return make_int2((int)(total * w / parts), (int)(total * (w + 1) / parts));
}
// Bits of `width` <= 64 tokens from position `base` on that drafted row i sees (bit t: token base + t), existing or not.
__device__ __forceinline__ unsigned long long sees(const TreeParams& p, int c0, int i, int d) {      // d = base - prefix
    const unsigned long long mask = p.masks ? (unsigned long long)p.masks[c0 + i] : ~0ull >> (63 - i);
    if (d >= 0) return d < 64 ? mask >> d : 0ull;
    if (d <= -64) return ~0ull;
    return (mask << -d) | ((1ull << -d) - 1ull);
}

// Host side, in tree_attn_sm100.cu.
int sm_count();
// The 128-row kernel (tree_attn_tile_sm100.cu).
int launch_tile(const TreeParams& p, int hd, bool fp8, int grid, cudaStream_t st);

}  // namespace tree
