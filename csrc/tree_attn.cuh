// Shared pieces of the tensor-core tree attention kernels (tree_attn_sm100.cu: tiles of 16 and 32 query rows on mma.sync,
// tree_attn_tile_sm100.cu: tiles of 128 rows on tcgen05): parameters, the cut of the work, the merge of partial results.
#pragma once
#include <cuda_fp8.h>

#include "tc.cuh"

typedef __nv_bfloat16 bf16;

namespace tree {

constexpr int PAGE = 16, MAX_B = 2048;

struct TreeParams {
    const bf16* q;
    long long q_stride;
    const uint8_t *ke, *ve;                            // exponents of 8-bit pages
    const int *table, *ctx_lens, *cu;
    const long long* masks;
    bf16* out;
    long long out_stride;
    float* part_o;                                     // [2 * grid][HD / 4][ROWS][4]
    float* part_ml;                                    // [2 * grid][ROWS][2]
    int* uoff;                                         // [B + 1] tiles before each sequence, for the merge kernel
    int max_pages, num_pages, B, N, H, G, n_kv, max_q, max_ctx;
    float scale_log2;
    int* status;
};

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// four e4m3 codes -> two f16 pairs
__device__ __forceinline__ void codes_to_f16(uint32_t c, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(c));
}
__device__ __forceinline__ float pow2_biased(int b) { return __uint_as_float(b > 0 ? (uint32_t)b << 23 : 0x00400000u); }
__device__ __forceinline__ void bulk_16(void* dst, const void* src, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(16), "r"(smem_u32(bar)) : "memory");
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

struct Segment {                                       // a CTA's part of one unit
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
// This block's part [lo, hi) of the line of tiles (empty where there are more blocks than tiles: every part that exists has a tile, since
// the merge reads all parts between a unit's first and last).
__device__ __forceinline__ int2 part_of_line(long long total) {
    const long long parts = min((long long)gridDim.x, total);
    if ((long long)blockIdx.x >= parts) return make_int2(0, 0);
    return make_int2((int)(total * blockIdx.x / parts), (int)(total * (blockIdx.x + 1) / parts));
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
int page_map(CUtensorMap* m, const void* base, long long rows, int hd, bool fp8, bool halves_apart);
// Puts the parts of the units together; `wide`: eight warps per row instead of one.
int merge(const TreeParams& p, int hd, int rows, int tile, int grid, bool wide, int zero_tail, cudaStream_t st);
// The 128-row kernel (tree_attn_tile_sm100.cu).
int launch_tile(const CUtensorMap& tmK, const CUtensorMap& tmV, const TreeParams& p, int hd, bool fp8, int grid, cudaStream_t st);

}  // namespace tree
