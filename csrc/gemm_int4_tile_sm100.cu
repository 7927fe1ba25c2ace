// Products with 4-bit weights for more than 16 tokens, on tcgen05: y[M, N] = x[M, K] . w[N, K]^T (+ c); see gemm_int4.cu for the weights.
//
// The weights are the 128-row operand, in tensor memory; up to 128 tokens are its columns, in shared memory.  Two blocks of 64 inputs are a turn
// (one group of 128, or two of 64).  Roles, a CTA per SM:
//
//   flush     4 or 8 warps: a group's sums from tensor memory times the row's scale (fp32), added to the row's sums in registers
//   widen     8 warps: 512 bytes of codes, copied ahead, -> 16 rows x 64 inputs as exact bf16 -> tensor memory
//   tokens    1 warp: x by TMA into the swizzled operand tile
//   issue     1 warp: eight products per turn
//
// Registers of the 16 x 256-bit store to tensor memory are (row r: columns 2 q, 2 q + 1), (row r + 8: the same), q = lane % 4: a word of codes expands
// into just that.  For step k lane q takes word q of the packed lane k of its row, so that the operand has the inputs in x's order.  The words are
// read from shared memory one by one; the copies' places there are exchanged (by the row's bits 1 and 2) so that no two meet in a bank.
//
// What bounds it: the length of a turn's way from codes to sums.  A turn of 64 tokens takes about 900 clocks, of which the products
// need 256: each role works 500 to 600 and waits for another the rest of the time, with the schedulers issuing in 54 % of the cycles (64 x 4096 x 14336:
// 18.2 us, of which the bytes would take 5.2).  At 1024 x 6144 x 4096 it reaches 910 TFLOP/s, 0.54 of the library's bf16 product, because
// every group's sums go through registers once.  Tried: x by 8-byte copies in the order that the store gives (30 us: issuing them), 16 widening warps
// (22 us), a barrier per operand (36 us at 64 x 28672 x 4096, 32 with one for both).  Weights widened into shared memory would move 48 KB through it
// per block, 384 clocks.
// Token tiles: up to 32, 64 or 128.  128 tokens x 6144 x 4096 take 14.5 us as one tile, 16.9 as two; 32 take 10.2 as a tile of 32, 11.6 of 64.
//
// Few row tiles: a cluster of up to eight CTAs shares the turns of a row tile and adds up through distributed shared memory, in
// the order of the ranks (64 x 4096 x 14336: 46 us without).  All waits are bounded (status word on timeout).
#include "attn_common.cuh"
#include "codes4.cuh"

typedef __nv_bfloat16 bf16;

namespace {

using namespace codes4;

constexpr int ROWS = 128, TURNS = 4, SCALES = 8;       // rows of a CTA, turns of operands (weights and tokens), groups of a flush thread's ring of scales
constexpr int D = 4;                                   // turns of a widening warp's ring
constexpr int PITCH = ROWS + 4;                        // floats of a token's sums

__device__ __forceinline__ void st_16x256_x4(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t ld_shared(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_peer(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int TN, int PG>
struct Roles {
    static constexpr int AC = TN > 64 ? 64 : 32;       // columns of a flush thread
    static constexpr int FLUSH = 4 * (TN / AC), WIDEN = 8, W_WIDEN = FLUSH, W_X = FLUSH + WIDEN, W_MMA = W_X + 1, THREADS = 32 * (W_MMA + 1);
    static constexpr int BLOCK = TN * 128;             // a block of 64 inputs of the tokens
    static constexpr int RING = TURNS * 2 * BLOCK, CODES = 8 * D * 2 * 512, SC = FLUSH * 32 * SCALES * 4;
    static constexpr int SMEM = 1024 + RING + CODES + SC;
    static constexpr int SETS = 2, SET = TN * (2 / PG);                // accumulators: sets, columns of a set (the groups of a turn)
    static_assert(TN * PITCH * 4 <= RING, "the partial sums take the ring's place");
    static_assert(TURNS * 64 + SETS * SET <= 512, "tensor memory");
};

template <int TN, int PG>
__global__ void __launch_bounds__(Roles<TN, PG>::THREADS, 1)
int4_tile_kernel(const __grid_constant__ CUtensorMap x, const uint4* packed, const bf16* scales, const bf16* c, bf16* y, int* status, int slices, const Shape s) {
    using R = Roles<TN, PG>;
    extern __shared__ uint8_t raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[TURNS], empty[TURNS], acc_full[R::SETS], acc_empty[R::SETS];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int slice = blockIdx.x % slices, n0 = blockIdx.x / slices * ROWS, m0 = blockIdx.y * TN;
    // this rank's turns (128 inputs each), its blocks
    const int all = (s.kb + 1) / 2, t0 = (int)((long long)all * slice / slices), turns = (int)((long long)all * (slice + 1) / slices) - t0;
    const int b0 = 2 * t0, nb = min(2 * turns, s.kb - b0);
    if (threadIdx.x == 0) {
        for (int i = 0; i < TURNS; ++i) {
            tc::mbar_init(&full[i], R::WIDEN + 1);     // (and the bytes of the tokens)
            tc::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < R::SETS; ++i) {
            tc::mbar_init(&acc_full[i], 1);
            tc::mbar_init(&acc_empty[i], R::FLUSH);
        }
        abort_word = 0;
        tc::fence_barrier_init();
    }
    if (warp == R::W_MMA) {
        tc::tmem_alloc(&tmem_slot, 512);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem_a = tmem_slot, tmem_acc = tmem_slot + TURNS * 64;
    float* part = reinterpret_cast<float*>(ring);                      // slices: [tokens][PITCH] sums, where the ring was
    bool ok = true;

    if (warp < R::FLUSH) {
        // ------------------------------------------------------------ sums of a group times the row's scale
        const int row = (warp & 3) * 32 + lane, tile = (n0 + row) >> 4, col0 = (warp >> 2) * R::AC;
        const bool live = tile < s.nt;
        const float unit = row & 8 ? UNIT1 : UNIT0;    // (of the sums, not of the scales: the largest of those times it would overflow)
        const uint32_t src = tmem_acc + ((uint32_t)((warp & 3) * 32) << 16) + col0;
        constexpr int G = 2 / PG, PIECE = R::AC > 32 ? 16 : 32;        // groups of a turn; columns of a load
        const int n_groups = PG == 2 ? turns : nb;
        // scales: the word of rows r and r + 8, a ring of this thread's own
        const bf16* sc = scales + ((long long)tile * s.ng + (PG == 2 ? t0 : b0)) * 16 + (row & 7) * 2;
        const uint32_t slots = smem_u32(ring + R::RING + R::CODES) + threadIdx.x * 4;
        auto fetch = [&](int g) {
            if (live && g < n_groups) copy4(slots + (g % SCALES) * (R::FLUSH * 128), sc + (long long)g * 16);
            copy_commit();
        };
#pragma unroll
        for (int i = 0; i < SCALES - 1; ++i) fetch(i);
        float2 acc[R::AC / 2];
#pragma unroll
        for (int i = 0; i < R::AC / 2; ++i) acc[i] = make_float2(0.f, 0.f);
        kb_dep_wait();
        kb_dep_trigger();
#pragma unroll 1
        for (int i = 0; i < turns; ++i) {
            const int set = i % R::SETS;
            float2 f[G];
#pragma unroll
            for (int h = 0; h < G; ++h) {
                const int g = i * G + h;
                copy_wait<SCALES - 2>();
                const uint32_t both = ld_shared(slots + (g % SCALES) * (R::FLUSH * 128));              // (rows that do not exist: anything)
                fetch(g + SCALES - 1);
                f[h].x = f[h].y = __uint_as_float(row & 8 ? both & 0xffff0000u : both << 16);
            }
            ok = tc::mbar_wait(&acc_full[set], (uint32_t)(i / R::SETS) & 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc::tc_fence_after();
            const bool both = G == 1 || i * G + 1 < n_groups;          // the last turn may have one group
#pragma unroll
            for (int h = 0; h < G; ++h) {
                if (h && !both) break;
#pragma unroll
                for (int e0 = 0; e0 < R::AC; e0 += PIECE) {
                    uint32_t v[PIECE];
                    if constexpr (PIECE == 32) tc::tmem_ld32(src + set * R::SET + h * TN + e0, v);
                    else tc::tmem_ld16(src + set * R::SET + h * TN + e0, v);
                    tc::tmem_ld_wait();
                    if (e0 + PIECE == R::AC && (h == G - 1 || !both)) {
                        tc::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&acc_empty[set]);
                    }
#pragma unroll
                    for (int e = 0; e < PIECE / 2; ++e)
                        acc[e0 / 2 + e] = __ffma2_rn(make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), f[h], acc[e0 / 2 + e]);
                }
            }
        }
        copy_wait<0>();
        if (!ok && lane == 0) atomicMax(status, (int)KB_TIMEOUT_EPI);
        const int n = n0 + row;
        if (slices > 1) {                              // (every product has read the ring: the last turn's sums were here)
#pragma unroll
            for (int i = 0; i < R::AC; ++i) part[(col0 + i) * PITCH + row] = (i & 1 ? acc[i / 2].y : acc[i / 2].x) * unit;
        } else if (n < s.N && ok) {
#pragma unroll
            for (int i = 0; i < R::AC; ++i) {
                const int m = m0 + col0 + i;
                if (m >= s.M) break;
                float v = (i & 1 ? acc[i / 2].y : acc[i / 2].x) * unit;
                if (c) v += __bfloat162float(c[(long long)m * s.c_stride + n]);
                y[(long long)m * s.y_stride + n] = __float2bfloat16(v);
            }
        }
    } else if (warp < R::W_X) {
        // ------------------------------------------------------------ codes -> operand
        constexpr int U = 2;                           // blocks of a turn
        const int w = warp - R::W_WIDEN, first = (w & 3) * 2 + (w >> 2);               // the tile's place among eight; a warp reaches lanes 32 (w % 4) ..
        const int r = lane >> 2, q = lane & 3, ex = r >> 1;
        constexpr int TURN = U * 512;                  // bytes of a turn: [block][32 lanes of 16]
        const uint32_t codes = smem_u32(ring + R::RING) + w * (D * TURN);
        const uint32_t put = codes + (lane ^ ex) * 16, get = codes + (4 * r + ex) * 16 + q * 4;        // ex: two bits, of the place in the row
        const uint4* src = packed + ((long long)min(n0 / 16 + first, s.nt - 1) * s.kb + b0) * 32 + lane;       // (rows behind the last: not stored)
        auto fetch = [&](int i) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i < turns && 2 * i + u < nb) copy16(put + (i % D) * TURN + u * 512, src + (long long)i * 64 + u * 32);
            copy_commit();
        };
#pragma unroll
        for (int i = 0; i < D - 1; ++i) fetch(i);
        kb_dep_wait();
        kb_dep_trigger();
#pragma unroll 1
        for (int i = 0; i < turns; ++i) {
            const int st = i % TURNS;
            copy_wait<D - 2>();
            __syncwarp();                              // the words are other lanes' copies; and all have read the turn that is filled next
            fetch(i + D - 1);
            const uint32_t at = get + (i % D) * TURN;
            uint32_t v[U][4], a[U][16];                // (of a block behind the last: what its place held, read by no product)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[u][k] = ld_shared((at ^ (k * 16)) + u * 512);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t e[4];
                    expand(v[u][k], e);
                    a[u][4 * k] = e[0];
                    a[u][4 * k + 1] = e[2];
                    a[u][4 * k + 2] = e[1];
                    a[u][4 * k + 3] = e[3];
                }
            ok = tc::mbar_wait(&empty[st], ((uint32_t)(i / TURNS) & 1u) ^ 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc::tc_fence_after();
            const uint32_t dst = tmem_a + st * 64 + ((uint32_t)(first * 16) << 16);
#pragma unroll
            for (int u = 0; u < U; ++u) st_16x256_x4(dst + u * 32, a[u]);
            tc::tmem_st_wait();
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&full[st]);
        }
        copy_wait<0>();
        if (!ok && lane == 0) atomicMax(status, (int)KB_TIMEOUT_TMA);
    } else if (warp == R::W_X) {
        // ------------------------------------------------------------ tokens (rows and inputs behind the last: zeros)
        kb_dep_wait();
        kb_dep_trigger();
        const bool lead = tc::elect_one();
#pragma unroll 1
        for (int i = 0; i < turns; ++i) {
            const int st = i % TURNS;
            ok = tc::mbar_wait(&empty[st], ((uint32_t)(i / TURNS) & 1u) ^ 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            if (lead) {
                const bool two = 2 * i + 1 < nb;
                const int k = (b0 + 2 * i) * KB;
                tc::mbar_expect_tx(&full[st], two ? 2 * R::BLOCK : R::BLOCK);
                tc::tma_load_3d(ring + st * 2 * R::BLOCK, &x, &full[st], k, m0, 0);
                if (two) tc::tma_load_3d(ring + (st * 2 + 1) * R::BLOCK, &x, &full[st], k + KB, m0, 0);
            }
            __syncwarp();
        }
        if (!ok && lane == 0) atomicMax(status, (int)KB_TIMEOUT_TMA);
    } else {
        // ------------------------------------------------------------ products
        kb_dep_wait();
        kb_dep_trigger();
        const uint32_t idesc = tc::instr_desc_f16(ROWS, TN, 1, 1, 0, 0);
        const tc::DescHalves d = tc::smem_desc_halves(smem_u32(ring), 16, 1024);
        const bool lead = tc::elect_one();
#pragma unroll 1
        for (int i = 0; i < turns; ++i) {
            const int st = i % TURNS, set = i % R::SETS;
            ok = tc::mbar_wait(&acc_empty[set], ((uint32_t)(i / R::SETS) & 1u) ^ 1u, abort_flag);
            ok = ok && tc::mbar_wait(&full[st], (uint32_t)(i / TURNS) & 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc::tc_fence_after();
            if (lead) {
                const uint32_t acc = tmem_acc + set * R::SET, a = tmem_a + st * 64, b = d.lo + ((st * 2 * R::BLOCK) >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) tc::mma_f16_ts_h(acc, a + 8 * k, b + 2 * k, d.hi, idesc, k != 0);
                if (2 * i + 1 < nb) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc::mma_f16_ts_h(acc + (PG == 1 ? TN : 0), a + 32 + 8 * k, b + (R::BLOCK >> 4) + 2 * k, d.hi, idesc, PG == 2 || k != 0);
                }
                tc::tc_commit(&empty[st]);
                tc::tc_commit(&acc_full[set]);
            }
            __syncwarp();
        }
        if (!ok && lane == 0) atomicMax(status, (int)KB_TIMEOUT_MMA);
    }

    if (slices > 1) {
        // ------------------------------------------------------------ sums of the ranks
        cluster_sync();
        const int cols = min(TN, s.M - m0);
        // rank q adds up the tokens q, q + slices, ..: four rows per thread, all ranks' sums on the way at once
        for (int i = threadIdx.x; i < (cols - slice + slices - 1) / slices * (ROWS / 4); i += R::THREADS) {
            const int t = slice + i / (ROWS / 4) * slices, row = i % (ROWS / 4) * 4, m = m0 + t;
            const uint32_t at = smem_u32(part + t * PITCH + row);
            float4 v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = q < slices ? ld_peer(peer_addr(at, q)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int q = 1; q < 8; ++q) {
                v[0].x += v[q].x;
                v[0].y += v[q].y;
                v[0].z += v[q].z;
                v[0].w += v[q].w;
            }
            const float sum[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = n0 + row + e;
                if (n < s.N) y[(long long)m * s.y_stride + n] = __float2bfloat16(sum[e] + (c ? __bfloat162float(c[(long long)m * s.c_stride + n]) : 0.f));
            }
        }
        cluster_sync();                                                // no CTA leaves while its sums are read
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == R::W_MMA) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem_a, 512);
    }
}

template <int TN, int PG>
int run(const bf16* x, const uint4* packed, const bf16* scales, const bf16* c, bf16* y, const Shape& s, int sms, int* status, cudaStream_t st) {
    using R = Roles<TN, PG>;
    static bool flags[64];
    bool* set = kb_device_flag(flags);
    if (!set) return 7;
    if (!*set) {
        if (cudaFuncSetAttribute(int4_tile_kernel<TN, PG>, cudaFuncAttributeMaxDynamicSharedMemorySize, R::SMEM) != cudaSuccess) return 7;
        *set = true;
    }
    attn::EncodeTiledFn enc = attn::get_encode();
    if (!enc) return 100;
    CUtensorMap map;
    const cuuint64_t dims[3] = {(cuuint64_t)s.K, (cuuint64_t)s.M, 1}, strides[2] = {(cuuint64_t)s.x_stride * 2, (cuuint64_t)s.M * s.x_stride * 2};
    const cuuint32_t box[3] = {KB, TN, 1}, estr[3] = {1, 1, 1};
    const CUresult r = enc(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<bf16*>(x), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return 200 + (int)r;
    const int tiles = (s.N + ROWS - 1) / ROWS, chunks = (s.M + TN - 1) / TN;
    if (chunks > 65535) return KB_BAD_ARG;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.blockDim = dim3(R::THREADS);
    cfg.dynamicSmemBytes = R::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    // as many ranks per row tile as run at once: a cluster lies within one group of SMs, so fewer fit than SMs / ranks
    static int fit[64][9];                             // [device][ranks]: clusters at once (0: not asked yet)
    int* mine = fit[set - flags];
    const long long units = (long long)tiles * chunks;
    int slices = units * 2 > sms ? 1 : (int)(sms / units);
    slices = slices > 8 ? 8 : slices;
    slices = slices > (s.kb + 1) / 2 ? (s.kb + 1) / 2 : slices;
    for (; slices > 1; --slices) {
        at[0].val.clusterDim.x = slices;
        cfg.gridDim = dim3(slices);
        cfg.numAttrs = 1;
        if (!mine[slices] && cudaOccupancyMaxActiveClusters(&mine[slices], int4_tile_kernel<TN, PG>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return KB_LAUNCH_FAILED;
        }
        if (units <= mine[slices]) break;
    }
    at[0].val.clusterDim.x = slices;
    cfg.gridDim = dim3(tiles * slices, chunks);
    cfg.numAttrs = g_kb_dependent_launch ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, int4_tile_kernel<TN, PG>, map, packed, scales, c, y, status, slices, s) != cudaSuccess) {
        cudaGetLastError();
        return KB_LAUNCH_FAILED;
    }
    return 0;
}

}  // namespace

int codes4::launch_tile(const bf16* x, const uint4* packed, const bf16* scales, const bf16* c, bf16* y, const Shape& s, int group, int sms, int* status,
                      cudaStream_t st) {
    if (s.M <= 32) return group == 64 ? run<32, 1>(x, packed, scales, c, y, s, sms, status, st) : run<32, 2>(x, packed, scales, c, y, s, sms, status, st);
    if (s.M <= 64) return group == 64 ? run<64, 1>(x, packed, scales, c, y, s, sms, status, st) : run<64, 2>(x, packed, scales, c, y, s, sms, status, st);
    // 128 tokens: two groups of 64 a turn, in two sets, would not fit tensor memory beside the weights
    return group == 64 ? run<64, 1>(x, packed, scales, c, y, s, sms, status, st) : run<128, 2>(x, packed, scales, c, y, s, sms, status, st);
}
