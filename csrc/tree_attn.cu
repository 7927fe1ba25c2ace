// Attention of drafted tokens over the paged cache, plain form: any head size in sixteens up to 256, bf16 or fp32 queries, pages of the
// queries' type or 8-bit pages (cache_fp8.cu).  A sequence's rows are the last of its cached tokens; a row sees every token in front
// of them and, of the rows themselves, those its mask names (bit j = row j), without masks the ones up to itself.
//
//   s_j = scale * q . k_j over the tokens j that the row sees,   o = sum_j softmax(s)_j v_j   (zero where it sees none)
//
// One block per (row, head): tiles of 128 tokens, one token per thread for the scores, one head dimension per thread for the
// output, an online softmax in fp32.  A token that is not seen is not read.  Compiled without fast-math.  The tensor-core form for
// heads of 64 and 128 in bf16 is tree_attn_sm100.cu.
#include <cuda_fp8.h>

#include "vec.cuh"

namespace {

constexpr int PAGE = 16, TILE = 128;

// Eight cached numbers as fp32.
template <typename T>
struct Rows {
    const T* p;
    __device__ __forceinline__ void load(long long row, int hd, int col, float* x) const { load8(p + row * hd + col, x); }
    __device__ __forceinline__ float one(long long row, int hd, int col) const { return to_float(p[row * hd + col]); }
};
struct Fp8Rows {
    const uint8_t *c, *e;
    __device__ __forceinline__ float factor(long long row) const {
        const uint32_t b = e[row];
        return __uint_as_float(b ? b << 23 : 0x00400000u);
    }
    __device__ __forceinline__ static float value(uint32_t code) {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
    }
    __device__ __forceinline__ void load(long long row, int hd, int col, float* x) const {
        const uint2 w = *reinterpret_cast<const uint2*>(c + row * hd + col);
        const float f = factor(row);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = value(((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 255u) * f;
    }
    __device__ __forceinline__ float one(long long row, int hd, int col) const { return value(c[row * hd + col]) * factor(row); }
};

struct TreeShape {
    int N, H, G, hd, B, max_pages, num_pages, max_q, max_ctx, zero_tail;
    long long q_stride, out_stride;
    float scale;
};

template <typename T, typename R>
__global__ void __launch_bounds__(TILE)
tree_plain_kernel(const T* __restrict__ q, const R kr, const R vr, const TreeShape s, const int* __restrict__ table,
                  const int* __restrict__ ctx_lens, const int* __restrict__ cu, const long long* __restrict__ masks, T* __restrict__ out,
                  int* __restrict__ status) {
    __shared__ float qs[256], ps[TILE], red[2][TILE / 32];
    __shared__ long long at[TILE];                     // cache row of every token of the tile, -1: not seen
    kb_dep_trigger();
    kb_dep_wait();
    const int n = blockIdx.x, head = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int kvh = head / (s.H / s.G);
    int b = n;
    if (cu) {
        int lo = 0, hi = s.B;                          // the sequence with cu[lo] <= n < cu[lo + 1]
        while (hi - lo > 1) {
            const int m = (lo + hi) >> 1;
            if (cu[m] <= n) lo = m; else hi = m;
        }
        b = lo;
    }
    T* dst = out + (long long)n * s.out_stride + (long long)head * s.hd;
    const int c0 = cu ? cu[b < s.B ? b : 0] : n, c1 = b < s.B ? (cu ? cu[b + 1] : n + 1) : n;
    if (b >= s.B || n < c0 || n >= c1) {               // behind the last sequence
        if (s.zero_tail)
            for (int d = t; d < s.hd; d += TILE) from_float(dst + d, 0.f);
        return;
    }
    const int rows = c1 - c0, ctx = ctx_lens[b];
    if (rows > s.max_q || rows > 64 || c1 > s.N || rows > ctx || ctx > s.max_ctx || (ctx + PAGE - 1) / PAGE > s.max_pages) {
        if (t == 0 && status) atomicMax(status, (int)KB_BAD_INDEX);
        for (int d = t; d < s.hd; d += TILE) from_float(dst + d, 0.f);
        return;
    }
    const int row = n - c0, prefix = ctx - rows;
    const unsigned long long sees = masks ? (unsigned long long)masks[n] : ~0ull >> (63 - row);
    for (int d = t; d < s.hd; d += TILE) qs[d] = to_float(q[(long long)n * s.q_stride + (long long)head * s.hd + d]) * s.scale;
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;  // dimensions t and t + 128
    __syncthreads();
    for (int t0 = 0; t0 < ctx; t0 += TILE) {
        const int tok = t0 + t, j = tok - prefix;
        float sc = -INFINITY;
        long long cell = -1;
        if (tok < ctx && (j < 0 || (sees >> j & 1ull))) {
            const int page = table[(long long)b * s.max_pages + tok / PAGE];
            if (page < 0 || page >= s.num_pages) {
                if (status) atomicMax(status, (int)KB_BAD_INDEX);
            } else {
                cell = ((long long)page * s.G + kvh) * PAGE + tok % PAGE;
                sc = 0.f;
                for (int c = 0; c < s.hd; c += 8) {
                    float x[8];
                    kr.load(cell, s.hd, c, x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) sc = fmaf(qs[c + i], x[i], sc);
                }
            }
        }
        float mx = warp_max(sc);
        if (lane == 0) red[0][warp] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;
        const float p = cell >= 0 ? expf(sc - base) : 0.f, f = expf(m - base);
        ps[t] = p;
        at[t] = cell;
        const float sum = warp_sum(p);
        if (lane == 0) red[1][warp] = sum;
        __syncthreads();
        l = l * f + (red[1][0] + red[1][1] + red[1][2] + red[1][3]);
        o0 *= f;
        o1 *= f;
        m = mn;
        const int cnt = min(TILE, ctx - t0);
        for (int i = 0; i < cnt; ++i) {
            if (at[i] < 0) continue;
            if (t < s.hd) o0 = fmaf(ps[i], vr.one(at[i], s.hd, t), o0);
            if (t + TILE < s.hd) o1 = fmaf(ps[i], vr.one(at[i], s.hd, t + TILE), o1);
        }
        __syncthreads();
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;        // l is NaN where a score was
    if (t < s.hd) from_float(dst + t, o0 * inv);
    if (t + TILE < s.hd) from_float(dst + t + TILE, o1 * inv);
}

}  // namespace

// q: [N, H, hd] in rows q_stride apart (type 0 = bf16, 1 = fp32); pages of that type, or codes with ke, ve non-null.  out: [N, H * hd] in
// rows out_stride apart.  cu null: row n is sequence n.  masks null: every row sees the rows up to itself.  zero_tail: rows behind the
// last sequence are set to zero, else left.
KB_API int kb_tree_attn_plain(const void* q, long long q_stride, const void* k, const void* ke, const void* v, const void* ve, const int* table,
                              int max_pages, int num_pages, const int* ctx_lens, const int* cu, int B, const long long* masks, void* out,
                              long long out_stride, int N, int H, int G, int hd, int max_q, int max_ctx, float scale, int zero_tail, int type,
                              int* status, cudaStream_t st) {
    if (N < 1 || H < 1 || H > 65535 || G < 1 || H % G || B < 1 || hd < 16 || hd > 256 || hd % 16 || max_pages < 1 || num_pages < 1 || max_q < 1 ||
        max_ctx < 1 || type < 0 || type > 1 || (ke == nullptr) != (ve == nullptr) || ((uintptr_t)k | (uintptr_t)v) % 16)
        return 5;
    const TreeShape s{N, H, G, hd, B, max_pages, num_pages, max_q, max_ctx, zero_tail, q_stride, out_stride, scale};
    const dim3 grid(N, H), block(TILE);
#define TREE_PLAIN(T, R, KR, VR)                                                                                                          \
    return kb_launch_dep(tree_plain_kernel<T, R>, grid, block, 0, st, (const T*)q, KR, VR, s, table, ctx_lens, cu, masks, (T*)out, status)
    if (ke) {
        const Fp8Rows kr{(const uint8_t*)k, (const uint8_t*)ke}, vr{(const uint8_t*)v, (const uint8_t*)ve};
        if (type == 0) TREE_PLAIN(bf16, Fp8Rows, kr, vr);
        TREE_PLAIN(float, Fp8Rows, kr, vr);
    }
    if (type == 0) TREE_PLAIN(bf16, Rows<bf16>, (Rows<bf16>{(const bf16*)k}), (Rows<bf16>{(const bf16*)v}));
    TREE_PLAIN(float, Rows<float>, (Rows<float>{(const float*)k}), (Rows<float>{(const float*)v}));
#undef TREE_PLAIN
}
