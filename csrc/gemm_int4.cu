// Products with 4-bit weights: y[M, N] = x[M, K] . w[N, K]^T (+ c), w[n, k] = scale[n, k / group] * (code[n, k] - 8), group 64 or 128.
//
// Mathematics.  Codes become bf16 numbers (code - 8) times a power of two, exactly (codes4.cuh).  The products of a group are summed in fp32 by
// the tensor cores, then times the group's scale in fp32 added to the result, so nothing is rounded but the result.
//
// Layout.  `mma.m16n8k16` with the weights as the 16-row operand and up to eight tokens as columns.  512 contiguous bytes are 16 rows x
// 64 inputs in the order of the fragments: a lane's 16 bytes hold, for the rows lane / 4 and lane / 4 + 8, the inputs 16 (lane % 4) .. + 15 of the
// block, four per word and k step - so the activations of a lane's fragments are 16 consecutive numbers of a row of x (the order of inputs
// inside a product is free as long as both operands have it).
//
// This file: up to 16 tokens (more: gemm_int4_tile_sm100.cu).  One block of threads per SM owns an even share of the row tiles; its warps share the
// groups of inputs and meet in shared memory once per step of up to four tiles.  Every warp streams its blocks - a block of each tile, the tokens' inputs
// for them, the scales - through a ring of its own by 16-byte asynchronous copies, across the steps, so that no load waits for arithmetic.
//
// What bounds it: no unit alone.  Of about 80 instructions per 512 bytes 36 widen the codes, 4 multiply; the rest is copies, addresses, sums.  At
// 8 x 28672 x 4096 the schedulers issue in 56 % of the cycles, the ALU is half busy, and 16 warps per SM do not cover the latencies in between (18 us,
// 3.4 TB/s; the 64 MB alone would take 9.5 us).  Tried: registers instead
// of the ring (23 us: fewer loads in flight), x straight from the L1 cache (27 us: it does not fit beside the rings), more and smaller
// blocks of threads (20 to 25 us), 8 warps (20 us).
#include <stddef.h>

#include "codes4.cuh"

typedef __nv_bfloat16 bf16;

namespace {

using namespace codes4;

__device__ __forceinline__ void mma_bf16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the first product of a sum
__device__ __forceinline__ void mma_bf16_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// the first `bytes` of 16, the others zero
__device__ __forceinline__ void copy16_part(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// TT tiles of eight tokens, RT tiles of 16 rows at once, PG blocks of 64 inputs per group, W warps, D stages of a warp's ring.
template <int TT, int RT, int W, int D>
struct Int4Smem {
    struct Stage {
        uint4 w[RT * 32];                              // a block of every row tile
        uint4 x[TT * 64];                              // its 64 inputs of the tokens: 16-byte chunk c of row r at c ^ (r & 7)
        uint32_t sc[RT * 8];
    } ring[W][D];
    float part[2][W][RT * 16][TT * 8 + 1];
};

template <int N>
struct Tiles {
    static constexpr int value = N;
};

// A block of threads owns an even share of the row tiles, taken up to RT at a time; its warps share the groups of inputs.
template <int TT, int RT, int PG, int W, int D>
__global__ void __launch_bounds__(W * 32, 1)
int4_kernel(const bf16* __restrict__ x, const uint4* __restrict__ packed, const uint32_t* __restrict__ scales, const bf16* c, bf16* y,
            const Shape s) {
    extern __shared__ __align__(16) unsigned char raw[];
    typedef Int4Smem<TT, RT, W, D> Smem;
    typedef typename Smem::Stage Stage;
    auto& sm = *reinterpret_cast<Smem*>(raw);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, qd = lane & 3, m0 = blockIdx.y * (TT * 8);
    const int t0 = (int)((long long)s.nt * blockIdx.x / gridDim.x), t1 = (int)((long long)s.nt * (blockIdx.x + 1) / gridDim.x);
    const int steps = (t1 - t0 + RT - 1) / RT, per = (t1 - t0 + steps - 1) / steps;
    // this warp's groups, in blocks: contiguous, so that it streams
    const int b0 = (int)((long long)s.ng * warp / W) * PG, b1 = min((int)((long long)s.ng * (warp + 1) / W) * PG, s.kb);
    const uint32_t ring = smem_u32(&sm.ring[warp][0]);

    // The copies run D - 1 blocks ahead.  Of the next: its block, its slot, the row tiles of its step, and this lane's addresses.
    struct At {
        int b, tile, cnt;
        uint32_t slot;
        const uint4* w;
        const uint32_t* sc;
    };
    const long long row_tile = (long long)s.kb * 32;
    auto enter = [&](At& at) {                         // the first block of a step
        at.b = b0;
        at.cnt = min(per, t1 - at.tile);
        at.w = packed + at.tile * row_tile + b0 * 32 + lane;
        at.sc = scales + ((long long)(at.tile + (lane >> 3)) * s.ng + b0 / PG) * 8 + (lane & 7);
    };
    auto next = [&](At& at) {
        at.slot = at.slot + sizeof(Stage) == ring + D * sizeof(Stage) ? ring : at.slot + (uint32_t)sizeof(Stage);
        ++at.b;
        at.w += 32;
        if (PG == 1 || at.b % PG == 0) at.sc += 8;
        if (at.b == b1) {
            at.tile += per;
            if (at.tile < t1) enter(at);
        }
    };
    auto copy_w = [&](const At& at) {
        const uint4* src = at.w;
#pragma unroll
        for (int t = 0; t < RT; ++t, src += row_tile)
            if (t == 0 || t < at.cnt) copy16(at.slot + t * 512 + lane * 16, src);
        if ((lane >> 3) < at.cnt) copy4(at.slot + offsetof(Stage, sc) + lane * 4, at.sc);
    };
    // x: lane -> rows lane / 8 + 4 i, chunk lane % 8; rows behind the last token are left as they are (their sums are not stored)
    const bf16* xp[TT * 2];
    bool there[TT * 2];
    uint32_t xdst[TT * 2];
#pragma unroll
    for (int i = 0; i < TT * 2; ++i) {
        const int row = (lane >> 3) + 4 * i;
        there[i] = m0 + row < s.M;
        xp[i] = x + (long long)(m0 + row) * s.x_stride + (lane & 7) * 8;
        xdst[i] = offsetof(Stage, x) + row * 128 + (((lane & 7) ^ row) & 7) * 16;
    }
    auto copy_x = [&](const At& at) {
        const bool in = at.b * KB + (lane & 7) * 8 < s.K;
#pragma unroll
        for (int i = 0; i < TT * 2; ++i)
            if (there[i]) copy16_part(at.slot + xdst[i], xp[i] + (in ? at.b * KB : 0), in ? 16 : 0);
    };
    At ahead;
    ahead.slot = ring;
    ahead.tile = b0 < b1 ? t0 : t1;
    if (b0 < b1) enter(ahead);
    // weights do not depend on the kernels ahead; activations and addends do
    {
        At at = ahead;
#pragma unroll
        for (int i = 0; i < D - 1; ++i)
            if (at.tile < t1) {
                copy_w(at);
                next(at);
            }
    }
    kb_dep_wait();
    kb_dep_trigger();
#pragma unroll
    for (int i = 0; i < D - 1; ++i) {
        if (ahead.tile < t1) {
            copy_x(ahead);
            next(ahead);
        }
        copy_commit();
    }
    int buf = 0;
    uint32_t slot = 0;
    for (int tile = t0; tile < t1; tile += per, buf ^= 1) {
        const int cnt = min(per, t1 - tile);
        float acc[RT][TT][4];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int j = 0; j < TT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][j][i] = 0.f;
        // T tiles of the step, without a branch among them
        auto walk = [&](auto tiles) {
            constexpr int T = decltype(tiles)::value;
#pragma unroll 1
            for (int b = b0; b < b1; b += PG) {
                float d[T][TT][4];
#pragma unroll
                for (int i = 0; i < PG; ++i) {
                    if (i && b + i >= b1) break;           // (then the last group has one block: b1 is the end of the row)
                    copy_wait<D - 2>();
                    __syncwarp();                          // the copies are all lanes'; and all have read the slot that is filled next
                    if (ahead.tile < t1) {
                        copy_w(ahead);
                        copy_x(ahead);
                        next(ahead);
                    }
                    copy_commit();
                    const Stage& st = *reinterpret_cast<const Stage*>(reinterpret_cast<const unsigned char*>(&sm.ring[warp][0]) + slot);
                    uint4 xb[TT][2];
#pragma unroll
                    for (int j = 0; j < TT; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h) xb[j][h] = st.x[(j * 8 + r) * 8 + ((2 * qd + h) ^ r)];
                    const bool last = i == PG - 1 || b + i + 1 == b1;
#pragma unroll
                    for (int t = 0; t < T; ++t) {
                        const uint4 v = st.w[t * 32 + lane];
                        uint32_t a[4];
                        expand(v.x, a);
#pragma unroll
                        for (int j = 0; j < TT; ++j)
                            if (i) mma_bf16(d[t][j], a, xb[j][0].x, xb[j][0].y);
                            else mma_bf16_first(d[t][j], a, xb[j][0].x, xb[j][0].y);
                        expand(v.y, a);
#pragma unroll
                        for (int j = 0; j < TT; ++j) mma_bf16(d[t][j], a, xb[j][0].z, xb[j][0].w);
                        expand(v.z, a);
#pragma unroll
                        for (int j = 0; j < TT; ++j) mma_bf16(d[t][j], a, xb[j][1].x, xb[j][1].y);
                        expand(v.w, a);
#pragma unroll
                        for (int j = 0; j < TT; ++j) mma_bf16(d[t][j], a, xb[j][1].z, xb[j][1].w);
                        if (last) {
                            const uint32_t sc = st.sc[t * 8 + r];
                            const float s0 = __uint_as_float(sc << 16), s1 = __uint_as_float(sc & 0xffff0000u);
#pragma unroll
                            for (int j = 0; j < TT; ++j)
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[t][j][e] = fmaf(e < 2 ? s0 : s1, d[t][j][e], acc[t][j][e]);
                        }
                    }
                    slot = slot == (D - 1) * sizeof(Stage) ? 0 : slot + (uint32_t)sizeof(Stage);
                }
            }
        };
        // a last step of fewer tiles than three: so many; else all, whatever the stage of one that is not there held before
        if (RT > 2 && cnt == 1) walk(Tiles<1>());
        else if (RT > 3 && cnt == 2) walk(Tiles<(RT > 2 ? 2 : 1)>());
        else walk(Tiles<RT>());
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                float* at = &sm.part[buf][warp][t * 16 + r][j * 8 + 2 * qd];
                at[0] = acc[t][j][0];
                at[1] = acc[t][j][1];
                at[8 * (TT * 8 + 1)] = acc[t][j][2];
                at[8 * (TT * 8 + 1) + 1] = acc[t][j][3];
            }
        }
        __syncthreads();                               // (the buffer of the step before is free: its readers have passed this barrier)
        for (int i = threadIdx.x; i < RT * 16 * TT * 8; i += W * 32) {
            const int row = i % (RT * 16), t = i / (RT * 16), n = tile * 16 + row, m = m0 + t;
            if (n >= s.N || row / 16 >= cnt || m >= s.M) continue;
            float v = 0.f;
#pragma unroll
            for (int q = 0; q < W; ++q) v += sm.part[buf][q][row][t];
            v *= row & 8 ? UNIT1 : UNIT0;
            if (c) v += __bfloat162float(c[(long long)m * s.c_stride + n]);
            y[(long long)m * s.y_stride + n] = __float2bfloat16(v);
        }
    }
    copy_wait<0>();
}

template <int TT, int RT, int PG, int W, int D>
int run_int4(const bf16* x, const uint4* packed, const uint32_t* scales, const bf16* c, bf16* y, const Shape& s, int ctas, cudaStream_t st) {
    const int chunks = (s.M + TT * 8 - 1) / (TT * 8);
    if (chunks > 65535) return 5;
    auto kernel = int4_kernel<TT, RT, PG, W, D>;
    const int bytes = sizeof(Int4Smem<TT, RT, W, D>);
    static bool done[64];
    bool* flag = kb_device_flag(done);
    if (flag == nullptr) return KB_LAUNCH_FAILED;
    if (!*flag && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return KB_LAUNCH_FAILED;
    *flag = true;
    const dim3 grid(s.nt < ctas ? s.nt : ctas, chunks);
    return kb_launch_dep(kernel, grid, dim3(W * 32), bytes, st, x, packed, scales, c, y, s);
}

}  // namespace

// x: [M, K] bf16 in rows x_stride apart (16-byte aligned rows), packed / scales as Int4Weight lays them out, c (may be null, may be y): [M, N].
KB_API int kb_gemm_int4(const void* x, long long x_stride, const void* packed, const void* scales, const void* c, long long c_stride, void* y,
                        long long y_stride, int M, int N, int K, int group, int* status, cudaStream_t st) {
    if (M < 1 || N < 1 || K < 8 || K % 8 || (group != 64 && group != 128) || x_stride % 8 || ((uintptr_t)x | (uintptr_t)packed) % 16 ||
        (uintptr_t)scales % 4)
        return 5;
    const Shape s{M, N, K, (N + 15) / 16, (K + KB - 1) / KB, (K + group - 1) / group, x_stride, y_stride, c_stride};
#define INT4_RUN(TT, RT, W, D)                                                                                                                \
    return group == 64 ? run_int4<TT, RT, 1, W, D>((const bf16*)x, (const uint4*)packed, (const uint32_t*)scales, (const bf16*)c, (bf16*)y, s, sms, st) \
                       : run_int4<TT, RT, 2, W, D>((const bf16*)x, (const uint4*)packed, (const uint32_t*)scales, (const bf16*)c, (bf16*)y, s, sms, st)
    // As many row tiles at once as a block owns, up to four: they share the tokens' copies, and a step ends in a barrier and sums over the warps.  us at
    // 8 tokens, K 4096, with 1 / 2 / 3 / 4 at once: N 4096 (two tiles a block) 5.8 / 4.9 / - / 4.9, N 6144 (three) 7.5 / 7.1 / 5.9 / 6.4, N 28672 (thirteen)
    // 25.3 / 20.2 / 18.6 / 18.0.  16 tokens: the second half of the columns doubles the copies; 12 and 8 warps leave room for three and four tiles.
    // More than 16 go to tcgen05: 16 tokens take 7.1 us here and 9.9 there at N 6144, 25 and 28 at N 28672; 32 tokens 13.3 and 10.2, 47 and 29.
    static int count[64];                              // SMs of each device, once asked
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 7;
    if (!count[dev] && cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 7;
    const int sms = count[dev];
    const int per = (s.nt + sms - 1) / sms;
    if (M <= 8) {
        if (per == 1) INT4_RUN(1, 1, 16, 3);
        if (per == 2) INT4_RUN(1, 2, 16, 3);
        if (per == 3 || per == 5 || per == 6) INT4_RUN(1, 3, 16, 3);
        INT4_RUN(1, 4, 16, 3);
    }
    if (M <= 16 || x_stride < K) {                     // (the other kernel's copies take rows that do not overlap)
        if (per <= 2) INT4_RUN(2, 2, 16, 3);
        if (per == 3 || per == 5 || per == 6) INT4_RUN(2, 3, 12, 3);
        INT4_RUN(2, 4, 8, 3);
    }
#undef INT4_RUN
    return launch_tile((const bf16*)x, (const uint4*)packed, (const bf16*)scales, (const bf16*)c, (bf16*)y, s, group, sms, status, st);
}
