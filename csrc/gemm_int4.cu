// Products with 4-bit weights: y[M, N] = x[M, K] . w[N, K]^T (+ c), w[n, k] = scale[n, k / group] * (code[n, k] - 8), group 64 or 128.
//
// Mathematics.  The codes enter the tensor cores as bf16 numbers 128 + c, which are one mask and one or of the packed word
// (0x4300 | nibble).  Per group the product is then  sum (128 + c) x = sum (c - 8) x + 136 sum x,  so the fp32 accumulator of a
// group starts at -136 * sum_{k in group} x and ends as sum (c - 8) x; it is scaled by the group's scale in fp32 and added to the result.
// The numbers are up to 32 times the ones that count, which costs five of the accumulator's 24 bits and no rounding of a
// weight: 2^-19 per group against the 2^-9 of the output.
//
// Layout.  `mma.m16n8k16` with the weights as the 16-row operand and up to eight tokens as columns.  512 contiguous bytes are 16 rows x
// 64 inputs in the order of the fragments: a lane's 16 bytes hold, for the rows lane / 4 and lane / 4 + 8, the inputs 16 (lane % 4) .. + 15 of the
// block, four per word and k step - so the activations of a lane's fragments are 16 consecutive numbers of a row of x, two
// 16-byte loads (the order of inputs inside a product is free as long as both operands have it).
#include "common.cuh"

typedef __nv_bfloat16 bf16;

namespace {

constexpr int KB = 64;                                 // inputs of a block

__device__ __forceinline__ void mma_bf16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One word (eight codes) -> the A fragment of one k step: pairs (row r, inputs 0 1), (r + 8, 0 1), (r, 2 3), (r + 8, 2 3), as 128 + code.
__device__ __forceinline__ void expand(uint32_t w, uint32_t* a) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
}

struct Int4Shape {
    int M, N, K, group, nt, kb, ng;
    long long x_stride, y_stride, c_stride;
};

constexpr int WARPS = 8;

// A block owns 16 rows of the weight and TT * 8 tokens; its warps share the K range, and their partial sums meet in shared memory.
template <int TT>
__global__ void __launch_bounds__(WARPS * 32)
int4_kernel(const bf16* __restrict__ x, const uint4* __restrict__ packed, const uint32_t* __restrict__ scales, const bf16* c, bf16* y,
            const Int4Shape s) {
    __shared__ float part[WARPS][16][TT * 8 + 1];
    kb_dep_trigger();
    kb_dep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, qd = lane & 3;
    const int tile = blockIdx.x, m0 = blockIdx.y * (TT * 8);
    float acc[TT][4];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
    const int per_group = s.group / KB;
    for (int g = warp; g < s.ng; g += WARPS) {
        float sum[TT], d[TT][4];
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            sum[t] = 0.f;
            d[t][0] = d[t][1] = d[t][2] = d[t][3] = 0.f;
        }
        for (int i = 0; i < per_group && g * per_group + i < s.kb; ++i) {
            const int blk = g * per_group + i, k0 = blk * KB + qd * 16;
            const uint4 w = packed[((long long)tile * s.kb + blk) * 32 + lane];
            uint32_t a[4][4];
            expand(w.x, a[0]);
            expand(w.y, a[1]);
            expand(w.z, a[2]);
            expand(w.w, a[3]);
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const int m = m0 + t * 8 + r;
                uint4 b[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                if (m < s.M) {
                    const bf16* px = x + (long long)m * s.x_stride + k0;
                    if (k0 < s.K) b[0] = *reinterpret_cast<const uint4*>(px);
                    if (k0 + 8 < s.K) b[1] = *reinterpret_cast<const uint4*>(px + 8);
                }
                float f[16];
                unpack8(*reinterpret_cast<const bf16x8*>(&b[0]), f);
                unpack8(*reinterpret_cast<const bf16x8*>(&b[1]), f + 8);
#pragma unroll
                for (int e = 0; e < 16; ++e) sum[t] += f[e];
                mma_bf16(d[t], a[0], b[0].x, b[0].y);
                mma_bf16(d[t], a[1], b[0].z, b[0].w);
                mma_bf16(d[t], a[2], b[1].x, b[1].y);
                mma_bf16(d[t], a[3], b[1].z, b[1].w);
            }
        }
        const uint32_t sc = scales[((long long)tile * s.ng + g) * 8 + r];
        const float s0 = __uint_as_float(sc << 16), s1 = __uint_as_float(sc & 0xffff0000u);
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            sum[t] += __shfl_xor_sync(0xffffffffu, sum[t], 1);
            sum[t] += __shfl_xor_sync(0xffffffffu, sum[t], 2);
            const float x0 = 136.f * __shfl_sync(0xffffffffu, sum[t], 8 * qd), x1 = 136.f * __shfl_sync(0xffffffffu, sum[t], 8 * qd + 4);
            acc[t][0] += s0 * (d[t][0] - x0);
            acc[t][1] += s0 * (d[t][1] - x1);
            acc[t][2] += s1 * (d[t][2] - x0);
            acc[t][3] += s1 * (d[t][3] - x1);
        }
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        part[warp][r][t * 8 + 2 * qd] = acc[t][0];
        part[warp][r][t * 8 + 2 * qd + 1] = acc[t][1];
        part[warp][r + 8][t * 8 + 2 * qd] = acc[t][2];
        part[warp][r + 8][t * 8 + 2 * qd + 1] = acc[t][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * TT * 8; i += WARPS * 32) {
        const int row = i & 15, t = i >> 4, n = tile * 16 + row, m = m0 + t;
        if (n >= s.N || m >= s.M) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += part[w][row][t];
        if (c) v += __bfloat162float(c[(long long)m * s.c_stride + n]);
        y[(long long)m * s.y_stride + n] = __float2bfloat16(v);
    }
}

}  // namespace

// x: [M, K] bf16 in rows x_stride apart (16-byte aligned rows), packed / scales as Int4Weight lays them out, c (may be null, may be y): [M, N].
KB_API int kb_gemm_int4(const void* x, long long x_stride, const void* packed, const void* scales, const void* c, long long c_stride, void* y,
                        long long y_stride, int M, int N, int K, int group, cudaStream_t st) {
    if (M < 1 || N < 1 || K < 8 || K % 8 || (group != 64 && group != 128) || x_stride % 8 || ((uintptr_t)x | (uintptr_t)packed) % 16 ||
        (uintptr_t)scales % 4)
        return 5;
    const Int4Shape s{M, N, K, group, (N + 15) / 16, (K + KB - 1) / KB, (K + group - 1) / group, x_stride, y_stride, c_stride};
    const int tokens = M <= 8 ? 8 : M <= 16 ? 16 : 32;
    const dim3 grid(s.nt, (M + tokens - 1) / tokens);
    if (grid.y > 65535) return 5;
#define INT4_RUN(TT)                                                                                                                   \
    return kb_launch_dep(int4_kernel<TT>, grid, dim3(WARPS * 32), 0, st, (const bf16*)x, (const uint4*)packed, (const uint32_t*)scales, \
                         (const bf16*)c, (bf16*)y, s)
    if (tokens == 8) INT4_RUN(1);
    if (tokens == 16) INT4_RUN(2);
    INT4_RUN(4);
#undef INT4_RUN
}
