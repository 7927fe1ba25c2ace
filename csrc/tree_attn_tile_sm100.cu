// Tree attention for many query rows per KV head (drafted tokens times query heads of the group): tiles of 128 rows x 128 cached tokens on
// tcgen05.  The work is cut as in tree_attn_sm100.cu (units of 128 rows, all units' tiles one line, equal parts, merge kernel); here a
// part is walked by one CTA per SM with a role per warp:
//
//   warps 0-7    softmax: two groups of four, group g has the tiles of parity g; one thread per row
//   warps 8-11   values: 8-bit pages -> f16 operand tile; places that hold no token -> zero.  Query rows -> shared memory, a unit ahead
//   warp 12      MMA issue (the whole warp walks the loop, one elected lane issues)
//   warps 13, 14 copies of keys and values, 16 bytes per lane
//   warp 15      what of a tile exists; 8-bit pages: factors of the keys, unit of the values
//
//   S = Q K^T    both operands K-major in shared memory, one accumulator per group
//                bf16 pages: kind::f16.  8-bit pages: kind::f8f6f4 on the codes as they lie in the cache; a query row, a power of two
//                taken out, is the sum of two e4m3 numbers, hi + lo, which together hold bf16's eight bits (down to 2^-9 of the row's
//                largest; below that the error is at most 2^-17 of the largest) - two products at twice the rate of one in 16 bits.
//   softmax      in fp32, a row at a time in one pass: exponentials against the maximum so far, which is renewed only when a
//                score exceeds it by more than 2^11 (2^20 where P is bf16); P back to tensor memory in 16 bits
//   O += P V     A = P in tensor memory, B = value tile in shared memory (MN-major), one accumulator per group, so that the groups
//                need nothing from one another before the end of a unit.  8-bit pages: P is f16 in units of 2^-4 (at most 2^15 with the
//                2^11 of lazy maxima: eleven bits down to 2^-18, off by at most 2^-29 below); the values' f16 carry the token's power
//                of two relative to E, the unit's largest so far (exact, since none lies below 2^(E - SPREAD)); O is in units of 2^(E - 6).
//                Values whose powers lie more than 2^SPREAD apart: as their codes, with a unit of O per row (apart_tile), so that a token
//                that a row does not see or gives no weight takes nothing from it, however large it is.  (64 rows over 131000 tokens: 245 us a call
//                without that code in the kernel, 251 with it, 2.5 times that where it runs; fp32 sums in its place 256 and 16 times.)
//
// The groups run out of step: one computes while the products of the other run.  Query rows are double-buffered by unit.
// Tokens that do not exist are masked in S and zeroed in the value tile (whatever the cache holds there).  Values of drafted tokens that
// are not finite must not meet the zero probabilities of rows that do not see them: such tokens are taken out of the value tile and
// added row by row (never in normal use).  All waits are bounded (status word on timeout).
#include "attn_common.cuh"
#include "tree_attn.cuh"

static_assert(tree::SPREAD <= 20, "factors of values are normal f16 numbers; codes times them are exact");

namespace {

using namespace tree;

constexpr int TT = 128, THREADS = 512;
constexpr int W_VAL = 8, W_MMA = 12, W_K = 13, W_V = 14, W_META = 15;
constexpr int SEGS = 16;                               // segments that the key warp may be ahead (it is less than eight tiles ahead)
constexpr int SLOTS = 8;                               // tiles that the notes on tiles reach ahead of the softmax, and more
constexpr int HALF = TT * 128;                         // 128 tokens x 128 bytes: 16 KB

template <bool FP8, int HD>
struct Lay {
    static constexpr int ROW_BYTES = FP8 ? HD : 2 * HD;
    static constexpr int HALVES = ROW_BYTES > 128 ? 2 : 1, ROWB = ROW_BYTES / HALVES;      // bytes of a staged row
    static constexpr int PIECE = TT * ROWB;            // one half of a staged tile
    static constexpr int KT = HALVES * PIECE;          // a staged tile of keys (or of values)
    static constexpr int VT = HD / 64 * HALF;          // a 16-bit value tile
    // stages of keys, of staged values, of value operand tiles (bf16: the staged tiles themselves)
    static constexpr int KST = 2, RST = FP8 ? 3 : 2, VST = 2;
    static constexpr int QT = FP8 ? 2 * KT : KT;       // query tile (8-bit pages: hi, lo)
    static constexpr int RING = KST * KT + RST * KT + (FP8 ? VST * VT : 0) + 2 * QT;
    static constexpr int EXPS = FP8 ? RST * 2 * TT : 0;
    static constexpr int FACT = FP8 ? SLOTS * TT * 4 : 0;
    static constexpr int ROWBUF = (FP8 ? 6 : 4) * TT * 4;
    static constexpr int VEXPS = FP8 ? SLOTS * TT : 0;
    static constexpr int SMEM = 1024 + RING + EXPS + FACT + ROWBUF + VEXPS;
};

__device__ __forceinline__ void mma_f8_h(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %2};\n\t"
        "mov.b64 db, {%3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc)
        : "memory");
}
// Whether a phase is over, without the suspension of a wait: the MMA warp mostly finds its barriers passed.
__device__ __forceinline__ bool passed(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ float2 f16x2_to_float(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }


// Columns of tensor memory (a row per lane) times f: fp32 accumulators, packed probabilities.
__device__ __noinline__ void scale_columns(uint32_t addr, int n, float f) {
#pragma unroll 1
    for (int c = 0; c < n; c += 32) {
        uint32_t o[32];
        tc::tmem_ld32(addr + c, o);
        tc::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
        tc::tmem_st32(addr + c, o);
    }
    tc::tmem_st_wait();
}
template <bool F16>
__device__ __noinline__ void scale_packed(uint32_t addr, int n, float f) {
    tc::tmem_st_wait();
#pragma unroll 1
    for (int c = 0; c < n; c += 16) {
        uint32_t o[16];
        tc::tmem_ld16(addr + c, o);
        tc::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 v = F16 ? f16x2_to_float(o[i]) : make_float2(__uint_as_float(o[i] << 16), __uint_as_float(o[i] & 0xffff0000u));
            o[i] = F16 ? pack_f16(v.x * f, v.y * f) : pack_bf16(v.x * f, v.y * f);
        }
        tc::tmem_st16(addr + c, o);
    }
    tc::tmem_st_wait();
}

constexpr int APART = -1;                              // for TileMeta::E: a unit per row, values as their codes
struct TileMeta {
    uint32_t valid[4], odd[4];                         // bits of the tile's tokens: exist; drafted with values that are not finite
    int E;                                             // 8-bit pages: biased exponent of the output's unit, or APART
};

// A tile's softmax with a unit of O per row, 2^D times that of the sums (SPREAD in tree_attn.cuh): probabilities carry their value's power
// of two relative to it.  The maximum m as it is, the sum l in units of 2^-SHIFT, by the threads of a warp, a row each.
struct RowState {
    float m, l, D;
};
template <int HD>
__device__ __noinline__ RowState apart_tile(uint32_t tmem_s, uint32_t tmem_o, const float* kf, const uint8_t* ev, unsigned long long seen0,
                                            unsigned long long seen1, float scale, bool begun, RowState st) {
    float mx = -INFINITY, y = -INFINITY;
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
        const uint32_t sees32 = (uint32_t)((q & 2 ? seen1 : seen0) >> (32 * (q & 1)));
        float x[32];
        tc::tmem_ld32(tmem_s + 32 * q, reinterpret_cast<uint32_t*>(x));
        tc::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const float v = sees32 >> i & 1u ? x[i] * kf[32 * q + i] * scale : -INFINITY;
            mx = fmaxf(mx, v);
            y = fmaxf(y, v + (float)((int)ev[32 * q + i] - 127));
        }
    }
    const float m = fmaxf(st.m, mx), at = m == -INFINITY ? 0.f : m;
    if (m != -INFINITY) st.l *= exp2f(st.m - m);
    const float D = fmaxf(st.D + (st.m - m), NO_UNIT), to = y - at > D + 11.f ? y - at - 4.f : D;      // (NaN: no maximum yet)
    if (begun && __any_sync(0xffffffffu, to != D)) scale_columns(tmem_o, HD, exp2f(D - to));
    float sum = 0.f;
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
        const uint32_t sees32 = (uint32_t)((q & 2 ? seen1 : seen0) >> (32 * (q & 1)));
        float x[32];
        tc::tmem_ld32(tmem_s + 32 * q, reinterpret_cast<uint32_t*>(x));
        tc::tmem_ld_wait();
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float p[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float a = sees32 >> (i + e) & 1u ? x[i + e] * kf[32 * q + i + e] * scale - at : -INFINITY;
                sum += exp2f(a);
                p[e] = exp2f(a + ((float)((int)ev[32 * q + i + e] - 127) - to));
            }
            pk[i >> 1] = pack_f16(p[0], p[1]);
        }
        tc::tmem_st16(tmem_s + 16 * q, pk);
    }
    tc::tmem_st_wait();
    return RowState{m, st.l + 16.f * sum, to};
}

template <bool FP8, int HD>
__global__ void __launch_bounds__(THREADS, 1)
tree_tile_kernel(const TreeParams p) {
    using L = Lay<FP8, HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sK = smem;
    uint8_t* sR = sK + L::KST * L::KT;                                 // staged values
    uint8_t* sV = FP8 ? sR + L::RST * L::KT : sR;                      // value operand tiles
    uint8_t* exps = smem + L::RING;                                    // [RST][2][TT] exponents of keys and values
    float* fact = reinterpret_cast<float*>(exps + L::EXPS);            // [SLOTS][TT] factors of scores, to log2 units
    uint8_t* sQ = smem + L::RING - 2 * L::QT;                          // two query tiles, staged like keys
    float* row_buf = reinterpret_cast<float*>(exps + L::EXPS + L::FACT);   // [2 groups][TT] maxima, then sums, then (8-bit pages) units of O
    uint8_t* vexps = exps + L::EXPS + L::FACT + L::ROWBUF;             // [SLOTS][TT] exponents of values, of tiles with a unit per row
    __shared__ int uoff[MAX_B + 1];
    __shared__ int wsum[THREADS / 32];
    __shared__ uint64_t k_full[L::KST], k_empty[L::KST], r_full[L::RST], r_empty[L::RST], v_ready[L::VST], f_ready[SLOTS], pv_done[L::VST], s_full[2], p_ready[2], q_ready[2],
        xch, slow[2];
    __shared__ uint32_t there[L::RST];                 // bit per page of the staged values: loaded
    __shared__ uint32_t there_k[SLOTS];                // the same of key tile j % SLOTS
    __shared__ TileMeta meta[SLOTS];                   // of tile j at j % SLOTS
    __shared__ uint32_t tmem_slot;
    __shared__ Segment segs[SEGS];
    __shared__ float q_scale[FP8 ? 2 * TT : 1];        // the power of two taken out of a query row
    __shared__ uint64_t seg_ready[SEGS];
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::KST; ++i) { tc::mbar_init(&k_full[i], 33); tc::mbar_init(&k_empty[i], 1); }
        for (int i = 0; i < L::RST; ++i) { tc::mbar_init(&r_full[i], 33); tc::mbar_init(&r_empty[i], 5); }
        for (int i = 0; i < L::VST; ++i) { tc::mbar_init(&v_ready[i], 4); tc::mbar_init(&pv_done[i], 1); }
        for (int i = 0; i < SLOTS; ++i) tc::mbar_init(&f_ready[i], 1);
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&s_full[i], 1);
            tc::mbar_init(&p_ready[i], 4);
            tc::mbar_init(&q_ready[i], 4);
            tc::mbar_init(&slow[i], 4);
        }
        for (int i = 0; i < SEGS; ++i) tc::mbar_init(&seg_ready[i], 1);
        tc::mbar_init(&xch, 8);
        abort_word = 0;
        tc::fence_barrier_init();
    }
    if (warp == W_MMA) {
        tc::tmem_alloc(&tmem_slot, 512);
        tc::tmem_relinquish();
    }
    kb_dep_wait();
    kb_dep_trigger();
    tc::tc_fence_before();
    count_tiles<TT, TT, THREADS>(p, uoff, wsum);       // (has the block's barriers)
    tc::tc_fence_after();
    const uint32_t tmem0 = tmem_slot, tmem_oacc = tmem0 + 256;             // S: two times 128 columns; O: two times HD
    const int2 part = part_of_line(uoff[p.B], blockIdx.x, gridDim.x);
    const int lo = part.x, n_tiles = part.y - part.x;
    bool ok = true;
    // The s-th segment of this part: found by the key warp, which is ahead of all others and a segment ahead of itself.
    auto segment = [&](int s) {
        Segment g;
        if (!tc::mbar_wait(&seg_ready[s % SEGS], (uint32_t)(s / SEGS) & 1u, abort_flag)) {
            ok = false;
            g.b = g.h = g.rb = g.t0 = 0;
            g.n = g.ctx = g.T = g.t1 = 1;
            return g;
        }
        return segs[s % SEGS];
    };

    if (n_tiles == 0) {
        // more blocks than tiles
    } else if (warp == W_K || warp == W_V) {
        // ------------------------------------------------------------ copies of keys, of values: 16 bytes per lane
        const bool isv = warp == W_V;
        // The key warp finds the segments, one ahead of the one that it works on (queries are fetched that early).
        int pub = 0, pub_at = 0;                       // segments published; tile at which the next one begins
        auto publish = [&]() {
            if (pub_at >= n_tiles) return;
            const Segment g = segment_at<TT, TT>(p, uoff, lo + pub_at, lo + n_tiles);
            if (lane == 0) {
                segs[pub % SEGS] = g;
                tc::mbar_arrive(&seg_ready[pub % SEGS]);
            }
            pub_at += g.t1 - g.t0;
            ++pub;
        };
        if (!isv) publish();
        Segment sg = segment(0);
        if (!isv) publish();
        int first = 0, seg = 0;                        // tile at which sg begins, its number
        int next = -2;                                 // lane l < 8: page l of the next tile (-2: behind the context)
        auto fetch = [&](int j) {
            if (j >= n_tiles) return;
            if (j - first >= sg.t1 - sg.t0) {
                sg = segment(++seg);
                first = j;
                if (!isv) publish();
            }
            const int tok = (sg.t0 + j - first) * TT + lane * PAGE;
            next = lane < 8 && tok < sg.ctx ? p.table[(long long)sg.b * p.max_pages + tok / PAGE] : -2;
        };
        fetch(0);
        for (int j = 0; j < n_tiles; ++j) {
            const int st = isv ? j % L::RST : j % L::KST, use = isv ? j / L::RST : j / L::KST;
            const bool good = next >= 0 && next < p.num_pages;
            if (next != -2 && !good && isv) atomicMax(p.status, (int)KB_BAD_INDEX);
            const long long mine = ((long long)next * p.n_kv + sg.h) * PAGE;       // first row of this lane's page
            const uint32_t have = __ballot_sync(0xffffffffu, good);
            fetch(j + 1);
            if (!ok) break;
            uint64_t* full = isv ? &r_full[st] : &k_full[st];
            if (isv && !FP8) {                         // the stage is the operand tile: free when its product has run
                if (use > 0) ok = tc::mbar_wait(&pv_done[st], (uint32_t)(use - 1) & 1u, abort_flag);
            } else {
                ok = tc::mbar_wait(isv ? &r_empty[st] : &k_empty[st], (uint32_t)(use & 1) ^ 1u, abort_flag);
            }
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            const uint8_t* src = (isv ? p.v : p.k) + lane * 16;
            const uint32_t dst = smem_u32((isv ? sR : sK) + st * L::KT);
#pragma unroll 1
            for (int pg = 0; pg < TT / PAGE; ++pg) {
                const long long row = __shfl_sync(0xffffffffu, mine, pg);
                if (!(have >> pg & 1u)) continue;
                const uint8_t* from = src + row * L::ROW_BYTES;
                const uint32_t to = dst + pg * PAGE * L::ROWB;
#pragma unroll
                for (int i = 0; i < PAGE * L::ROW_BYTES / 512; ++i) {
                    const int q = i * 32 + lane;       // 16-byte piece of the page: its row, half and swizzled place
                    const int t = q / (L::ROW_BYTES / 16), c = q % (L::ROW_BYTES / 16), h = c / (L::ROWB / 16), cc = c % (L::ROWB / 16);
                    copy16(to + h * L::PIECE + t * L::ROWB + ((cc ^ (L::ROWB == 128 ? t & 7 : (t >> 1) & 3)) << 4), from + i * 512);
                }
            }
            if (FP8 && isv && lane < 16) {             // exponents of the keys, then of the values
                const long long row = __shfl_sync(0xffffu, mine, lane & 7);
                if (have >> (lane & 7) & 1u)
                    copy16(smem_u32(exps + st * 2 * TT + (lane >> 3) * TT + (lane & 7) * PAGE), (lane < 8 ? p.ke : p.ve) + row);
            }
            copy_arrive(full);
            if (lane == 0) {
                if (isv) there[st] = have;
                else there_k[j % SLOTS] = have;
                tc::mbar_arrive(full);
            }
        }
        copy_wait<0>();                                // copies in flight land before the block can exit
        if (!ok && lane == 0) atomicMax(p.status, (int)KB_TIMEOUT_TMA);
    } else if (warp == W_MMA) {
        // ------------------------------------------------------------ products
        const uint32_t id_s = FP8 ? (1u << 4) | (uint32_t)(TT >> 3) << 17 | (uint32_t)(TT >> 4) << 24 : tc::instr_desc_f16(TT, TT, 1, 1, 0, 0);
        const uint32_t id_o = tc::instr_desc_f16(TT, HD, FP8 ? 0 : 1, FP8 ? 0 : 1, 0, 1);
        tc::DescHalves dk = tc::smem_desc_halves(smem_u32(sK), 16, L::ROWB * 8), dq = tc::smem_desc_halves(smem_u32(sQ), 16, L::ROWB * 8);
        if (L::ROWB == 64) dq.hi = dk.hi = (dk.hi & ~(7u << 29)) | 4u << 29;       // rows of 64 bytes: 64-byte swizzle
        const tc::DescHalves dv = tc::smem_desc_halves(smem_u32(sV), HALF, 1024);
        Segment sg = segment(0);
        const int len0 = sg.t1 - sg.t0;
        int s_left = len0, s_seg = 0;                  // tiles of the segment that S is at; its number
        bool s_new = true;                             // its queries have not been waited for
        auto wait = [&](uint64_t* bar, uint32_t parity) { return passed(bar, parity) || tc::mbar_wait(bar, parity, abort_flag); };
        auto scores = [&](int j) {                     // S(j): waits for its queries and keys
            if (s_left == 0) {
                sg = segment(++s_seg);
                if (!ok) return false;
                s_left = sg.t1 - sg.t0;
                s_new = true;
            }
            --s_left;
            const int st = j % L::KST;
            if (s_new && !wait(&q_ready[s_seg & 1], (uint32_t)(s_seg >> 1) & 1u)) return false;
            s_new = false;
            if (!wait(&k_full[st], (uint32_t)(j / L::KST) & 1u)) return false;
            tc::fence_proxy_async();                   // the keys were copied through the generic proxy
            tc::tc_fence_after();
            const uint32_t b_lo = dk.lo + st * (L::KT >> 4), a_lo = dq.lo + (s_seg & 1) * (L::QT >> 4), d = tmem0 + (j & 1) * 128;
            if (tc::elect_one()) {
                if constexpr (FP8) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int k = 0; k < HD / 32; ++k)
                            mma_f8_h(d, a_lo + ((i * L::KT + k * 32) >> 4), dq.hi, b_lo + (k * 32 >> 4), dk.hi, id_s, (i | k) != 0);
                } else {
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint32_t off = ((k >> 2) * HALF + (k & 3) * 32) >> 4;
                        tc::mma_f16_h(d, a_lo + off, dq.hi, b_lo + off, dk.hi, id_s, k != 0);
                    }
                }
                tc::tc_commit(&s_full[j & 1]);
                tc::tc_commit(&k_empty[st]);
            }
            __syncwarp();
            return true;
        };
        int o_at = 0, o_len = len0, o_seg = 0;         // tile of the segment that O is at; its number
        ok = ok && scores(0) && (n_tiles < 2 || scores(1));
        for (int j = 0; j < n_tiles && ok; ++j) {
            if (o_at == o_len) {
                const Segment og = segment(++o_seg);
                if (!ok) break;
                o_len = og.t1 - og.t0;
                o_at = 0;
            }
            const int vs = j % L::VST;
            ok = wait(&v_ready[vs], (uint32_t)(j / L::VST) & 1u) && wait(&p_ready[j & 1], (uint32_t)(j >> 1) & 1u);
            if (!ok) break;
            if (!FP8) tc::fence_proxy_async();         // (8-bit pages: the warps that wrote the operand have fenced)
            tc::tc_fence_after();
            // a group's first tile overwrites its O, unless the softmax warps have begun it (values that are not finite)
            const TileMeta& mt = meta[j % SLOTS];
            const uint32_t acc = o_at > 1 || (mt.odd[0] | mt.odd[1] | mt.odd[2] | mt.odd[3]) ? 1u : 0u;
            const uint32_t b_lo = dv.lo + vs * (L::VT >> 4), a = tmem0 + (j & 1) * 128;
            if (tc::elect_one()) {
#pragma unroll
                for (int k = 0; k < TT / 16; ++k) tc::mma_f16_ts_h(tmem_oacc + (j & 1) * HD, a + 8 * k, b_lo + (k * 2048 >> 4), dv.hi, id_o, k == 0 ? acc : 1u);
                tc::tc_commit(&pv_done[vs]);
            }
            __syncwarp();
            ++o_at;
            if (j + 2 < n_tiles) ok = scores(j + 2);
        }
        if (!ok && lane == 0) atomicMax(p.status, (int)KB_TIMEOUT_MMA);
    } else if (warp == W_META) {
        // ------------------------------------------------------------ what of a tile exists, which drafted tokens are odd, factors
        Segment sg = segment(0);
        int first = 0, seg = 0;                        // tile at which sg begins, its number
        uint32_t E = 0, low = 255;
        for (int j = 0; j < n_tiles; ++j) {
            if (j - first == sg.t1 - sg.t0) {
                sg = segment(++seg);
                first = j;
            }
            if (!ok) break;
            const int rst = j % L::RST;
            // (slot j % SLOTS is free: the load of tile j waited for the conversion, and with it the product, of tiles less than SLOTS back)
            ok = tc::mbar_wait(&r_full[rst], (uint32_t)(j / L::RST) & 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            const int base = (sg.t0 + j - first) * TT, prefix = sg.ctx - sg.n;
            const uint32_t have = there[rst];
            const bool edge = have != 0xffu || base + TT > prefix;
            const uint8_t* e = exps + rst * 2 * TT;
            TileMeta& mt = meta[j % SLOTS];
            uint32_t top = 0, bot = 255;
#pragma unroll
            for (int w = 0; w < 4; ++w) {              // 32 tokens at a time
                const int t = w * 32 + lane, tok = base + t;
                const bool valid = !edge || (tok < sg.ctx && (have >> (t / PAGE) & 1u));
                if constexpr (FP8) {
                    fact[(j % SLOTS) * TT + t] = pow2_biased(e[t]) * p.scale_log2;
                    const uint32_t ev = e[TT + t];
                    if (valid && ev != 255u) {
                        top = max(top, ev);
                        bot = min(bot, ev);
                    }
                }
                uint32_t vword = 0xffffffffu, oword = 0u;
                if (edge) {
                    vword = __ballot_sync(0xffffffffu, valid);
                    const uint8_t* raw = sR + rst * L::KT + t * L::ROWB;
                    bool bad = false;
                    if (valid && tok >= prefix)
                        for (int h = 0; h < L::HALVES; ++h)
                            for (int c = 0; c < L::ROWB / 16; ++c) {
                                const uint4 v = *reinterpret_cast<const uint4*>(raw + h * L::PIECE + c * 16);
                                const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int q = 0; q < 4; ++q)
                                    bad |= FP8 ? __vcmpeq4(x[q] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0u : __vcmpeq2(x[q] & 0x7f807f80u, 0x7f807f80u) != 0u;
                            }
                    oword = __ballot_sync(0xffffffffu, bad);
                }
                if (lane == 0) {
                    mt.valid[w] = vword;
                    mt.odd[w] = oword;
                }
            }
            if constexpr (FP8) {                       // the unit of the output: largest exponent of the unit's values so far
                top = __reduce_max_sync(0xffffffffu, top);
                bot = __reduce_min_sync(0xffffffffu, bot);
                E = j == first ? top : max(E, top);
                low = j == first ? bot : min(low, bot);
                const bool apart = (int)E - (int)low > SPREAD;
                if (lane == 0) mt.E = apart ? APART : (int)E;
                if (apart)
#pragma unroll
                    for (int w = 0; w < 4; ++w) vexps[(j % SLOTS) * TT + w * 32 + lane] = e[TT + w * 32 + lane];
            }
            __syncwarp();
            if (lane == 0) {
                tc::mbar_arrive(&f_ready[j % SLOTS]);
                if (FP8) tc::mbar_arrive(&r_empty[rst]);
            }
        }
        if (!ok && lane == 0) atomicMax(p.status, (int)KB_TIMEOUT_TMA);
    } else if (warp >= W_VAL) {
        // ------------------------------------------------------------ values: thread = token of the tile, and = query row
        const int t = threadIdx.x - W_VAL * 32;
        auto load_queries = [&](const Segment& sg, int seg) {
            const int R = sg.rb * TT + t;
            const bool live = R < sg.n * p.G;
            const bf16* src = p.q + (long long)((p.cu ? p.cu[sg.b] : sg.b) + (live ? R / p.G : 0)) * p.q_stride + (long long)(sg.h * p.G + (live ? R % p.G : 0)) * HD;
            uint8_t* dst = sQ + (seg & 1) * L::QT + t * L::ROWB;
            const int sw = L::ROWB == 128 ? t & 7 : (t >> 1) & 3;
            uint4 v[HD / 8];
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) v[i] = live ? *reinterpret_cast<const uint4*>(src + i * 8) : make_uint4(0u, 0u, 0u, 0u);
            if constexpr (FP8) {
                uint32_t big = 0;
#pragma unroll
                for (int i = 0; i < HD / 8; ++i) big = max(big, max(max(largest(v[i].x), largest(v[i].y)), max(largest(v[i].z), largest(v[i].w))));
                const float inv = q_down(big);
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) {    // sixteen numbers: a chunk of hi, a chunk of lo
                    uint4 h4, l4;
                    split_e4m3(make_uint2(v[2 * c].x, v[2 * c].y), inv, h4.x, l4.x);
                    split_e4m3(make_uint2(v[2 * c].z, v[2 * c].w), inv, h4.y, l4.y);
                    split_e4m3(make_uint2(v[2 * c + 1].x, v[2 * c + 1].y), inv, h4.z, l4.z);
                    split_e4m3(make_uint2(v[2 * c + 1].z, v[2 * c + 1].w), inv, h4.w, l4.w);
                    *reinterpret_cast<uint4*>(dst + ((c ^ sw) << 4)) = h4;
                    *reinterpret_cast<uint4*>(dst + L::KT + ((c ^ sw) << 4)) = l4;
                }
                q_scale[(seg & 1) * TT + t] = q_up(big);
            } else {
#pragma unroll
                for (int c = 0; c < HD / 8; ++c) *reinterpret_cast<uint4*>(dst + (c >> 3) * HALF + (((c & 7) ^ sw) << 4)) = v[c];
            }
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&q_ready[seg & 1]);
        };
        Segment sg = segment(0);
        int at = 0, seg = 0, loaded = 0;               // tile within the segment, its number; segments whose queries are loaded
        for (int j = 0; j < n_tiles; ++j, ++at) {
            const int vs = j % L::VST, rst = j % L::RST;
            if (at == sg.t1 - sg.t0) {
                sg = segment(++seg);
                at = 0;
            }
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            // queries of this unit, or of the next one once the products of the unit before this one (the buffer's last reader) have run
            const bool ahead = at == 1 && loaded == seg + 1 && j - at + (sg.t1 - sg.t0) < n_tiles;
            if (loaded <= seg || ahead) {
                if (j >= 2) ok = tc::mbar_wait(&pv_done[(j - 2) % L::VST], (uint32_t)((j - 2) / L::VST) & 1u, abort_flag);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                if (loaded <= seg) {
                    load_queries(sg, seg);
                    loaded = seg + 1;
                } else {
                    load_queries(segment(seg + 1), seg + 1);
                    loaded = seg + 2;
                }
            }
            ok = tc::mbar_wait(&f_ready[j % SLOTS], (uint32_t)(j / SLOTS) & 1u, abort_flag);
            // the operand stage is free when the product two tiles back has run
            if (FP8 && ok && j >= 2) ok = tc::mbar_wait(&pv_done[vs], (uint32_t)((j - 2) / L::VST) & 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            const TileMeta& mt = meta[j % SLOTS];
            const uint32_t vword = mt.valid[warp - W_VAL];
            uint8_t* op = sV + vs * L::VT;
            if constexpr (FP8) {
                // the token's factor, an f16 power of two from 2^(6 - SPREAD) to 2^6 (twice); none where the probabilities carry it
                const uint8_t* raw = sR + rst * L::KT;
                const int ev = exps[rst * 2 * TT + TT + t], w = ev == 255 || mt.E == APART ? 0 : ev - mt.E + 6;
                const uint32_t one = vword >> lane & 1u ? (uint32_t)(w + 15) << 10 : 0u;
                const uint32_t mine = one | one << 16;
                // codes -> f16: a warp takes whole rows, 16 codes per lane, so that loads and stores use all banks
                constexpr int CH = HD / 16, RPW = 32 / CH;     // chunks per row, rows per warp step
                const int c = lane % CH;
                constexpr int U = 4;                           // rows in flight
#pragma unroll 1
                for (int i0 = 0; i0 < 32 / RPW; i0 += U) {
                    uint4 v[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int row = (warp - W_VAL) * 32 + (i0 + u) * RPW + lane / CH;
                        v[u] = *reinterpret_cast<const uint4*>(raw + row * L::ROWB + ((c ^ (HD == 128 ? row & 7 : (row >> 1) & 3)) << 4));
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int row = (warp - W_VAL) * 32 + (i0 + u) * RPW + lane / CH;
                        const uint32_t f = __shfl_sync(0xffffffffu, mine, row & 31);
                        if (!(vword >> (row & 31) & 1u)) v[u] = make_uint4(0u, 0u, 0u, 0u);
                        uint4 a, b;
                        codes_to_f16(v[u].x, a.x, a.y);
                        codes_to_f16(v[u].y, a.z, a.w);
                        codes_to_f16(v[u].z, b.x, b.y);
                        codes_to_f16(v[u].w, b.z, b.w);
                        a = make_uint4(mul_f16x2(a.x, f), mul_f16x2(a.y, f), mul_f16x2(a.z, f), mul_f16x2(a.w, f));
                        b = make_uint4(mul_f16x2(b.x, f), mul_f16x2(b.y, f), mul_f16x2(b.z, f), mul_f16x2(b.w, f));
                        uint8_t* dst = op + (c >> 2) * HALF + row * 128;
                        const int c0 = (c & 3) * 2, flip = (c >> 2) & 1;   // the two halves of a row share banks: store them in opposite order
                        *reinterpret_cast<uint4*>(dst + (((c0 + flip) ^ (row & 7)) << 4)) = flip ? b : a;
                        *reinterpret_cast<uint4*>(dst + (((c0 + 1 - flip) ^ (row & 7)) << 4)) = flip ? a : b;
                    }
                }
                tc::fence_proxy_async();
            } else if (vword != 0xffffffffu) {
                if (!(vword >> lane & 1u))
#pragma unroll
                    for (int h = 0; h < L::HALVES; ++h)
                        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(op + h * HALF + t * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                tc::fence_proxy_async();
            }
            __syncwarp();
            if (lane == 0) {
                tc::mbar_arrive(&v_ready[vs]);
                if (FP8) tc::mbar_arrive(&r_empty[rst]);
            }
        }
        if (!ok && lane == 0) atomicMax(p.status, (int)KB_TIMEOUT_TMA);
    } else {
        // ------------------------------------------------------------ softmax: a thread per row, tiles of parity g
        const int g = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem0 + g * 128 + lane_base, tmem_o = tmem_oacc + g * HD + lane_base;
        uint32_t n_slow = 0, n_x = 0;
        auto exchange = [&](uint64_t* bar, uint32_t& count) {
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar);
            const bool good = tc::mbar_wait(bar, count & 1u, abort_flag);
            ++count;
            return good;
        };
        // log2 units: the maximum is renewed when a score exceeds it by more than GROW; P is in units of 2^-SHIFT.  f16 holds 2^(GROW + SHIFT)
        constexpr float GROW = FP8 ? 11.f : 20.f, SHIFT = FP8 ? 4.f : 0.f;
        int j0 = 0;
        for (int seg = 0; j0 < n_tiles && ok; ++seg) {
            const Segment sg = segment(seg);
            if (!ok) break;
            const int len = sg.t1 - sg.t0, M = sg.n * p.G, R = sg.rb * TT + r, c0 = p.cu ? p.cu[sg.b] : sg.b, prefix = sg.ctx - sg.n;
            const bool live = sg.rb * TT + (warp & 3) * 32 < M;            // the warp has rows
            const int row_i = min(R, M - 1) / p.G, row_g = min(R, M - 1) % p.G;
            float scale = FP8 ? 1.f : p.scale_log2;        // 8-bit pages: the row's power of two, which rounds nothing
            // A group without a tile of the segment does not wait for its queries: it could come so late that the queries two segments on have
            // turned the barrier's parity once more (they are loaded when the segment's products have run, for which only groups with a tile
            // are needed)
            if (FP8 && (len > 1 || g == (j0 & 1))) {
                if (!tc::mbar_wait(&q_ready[seg & 1], (uint32_t)(seg >> 1) & 1u, abort_flag)) { ok = false; break; }
                scale = q_scale[(seg & 1) * TT + r];
            }
            float m_used = -INFINITY, l = 0.f;
            int E = 0;
            constexpr int OWN = -2;                    // for E: O is in units of 2^D times that of the sums, not of 2^(E - 137)
            float& D = row_buf[(FP8 ? 4 + g : 0) * TT + r];        // (E == OWN)
            bool begun = false;                        // the group has had a tile of this segment
            for (int at = (g ^ j0) & 1; at < len; at += 2) {
                const int j = j0 + at, vs = j % L::VST, base = (sg.t0 + at) * TT;
                if (!tc::mbar_wait(&s_full[g], (uint32_t)(j >> 1) & 1u, abort_flag)) { ok = false; break; }
                tc::tc_fence_after();
                // tiles with drafted tokens, with the end of the context, or with pages that are not there
                const bool edge = base + TT > prefix || there_k[j % SLOTS] != 0xffu;
                if ((FP8 || edge) && !tc::mbar_wait(&f_ready[j % SLOTS], (uint32_t)(j / SLOTS) & 1u, abort_flag)) { ok = false; break; }
                const TileMeta& mt = meta[j % SLOTS];
                uint32_t odd_any = 0;
                unsigned long long seen[2] = {~0ull, ~0ull};
                if (edge) {
                    odd_any = mt.odd[0] | mt.odd[1] | mt.odd[2] | mt.odd[3];
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf)
                        seen[hf] = sees(p, c0, row_i, base + hf * 64 - prefix) &
                                   ((unsigned long long)mt.valid[2 * hf] | (unsigned long long)mt.valid[2 * hf + 1] << 32);
                }
                if (live) {
                    const float* kf = fact + (j % SLOTS) * TT;
                    const int E_new = FP8 ? mt.E : 0;
                    int q0 = 0;
                    if (FP8 && E_new != E) {
                        if (E_new == APART) {
                            if (E != OWN) D = begun ? (float)(E - 137) : NO_UNIT;
                            const RowState rs = apart_tile<HD>(tmem_s, tmem_o, kf, vexps + (j % SLOTS) * TT, seen[0], seen[1], scale, begun,
                                                               RowState{m_used, l, D});
                            m_used = rs.m;
                            l = rs.l;
                            D = rs.D;
                            E = OWN;
                            q0 = 4;
                        } else {
                            if (begun) scale_columns(tmem_o, HD, exp2f((float)(E - E_new)));
                            E = E_new;
                        }
                    }
                    const float2 sc2 = make_float2(scale, scale);
                    float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    // 32 columns at a time.  The loop stays rolled: unrolled, the instruction cache is what bounds this kernel
#pragma unroll 1
                    for (int q = q0; q < 4; ++q) {
                        float x[32];
                        tc::tmem_ld32(tmem_s + 32 * q, reinterpret_cast<uint32_t*>(x));
                        tc::tmem_ld_wait();
                        if constexpr (FP8) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const float4 f = *reinterpret_cast<const float4*>(kf + 32 * q + i);
                                const float2 u = __fmul2_rn(make_float2(x[i], x[i + 1]), make_float2(f.x, f.y));
                                const float2 v = __fmul2_rn(make_float2(x[i + 2], x[i + 3]), make_float2(f.z, f.w));
                                x[i] = u.x;
                                x[i + 1] = u.y;
                                x[i + 2] = v.x;
                                x[i + 3] = v.y;
                            }
                        } else {                       // (before anything is hidden or subtracted: see tree_attn_sm100.cu)
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 u = __fmul2_rn(make_float2(x[i], x[i + 1]), sc2);
                                x[i] = u.x;
                                x[i + 1] = u.y;
                            }
                        }
                        const uint32_t sees32 = (uint32_t)(seen[q >> 1] >> (32 * (q & 1)));
                        if (edge) {                    // what is not seen
#pragma unroll
                            for (int i = 0; i < 32; ++i) x[i] = sees32 >> i & 1u ? x[i] : -INFINITY;
                        }
                        float m4[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) m4[i] = attn::fmax3(x[3 * i], x[3 * i + 1], x[3 * i + 2]);
#pragma unroll
                        for (int i = 12; i < 28; i += 8) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) m4[e] = attn::fmax3(m4[e], x[i + 2 * e], x[i + 2 * e + 1]);
                        }
                        m4[0] = attn::fmax3(m4[0], x[28], x[29]);
                        m4[1] = attn::fmax3(m4[1], x[30], x[31]);
                        const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * (FP8 ? scale : 1.f);
                        if (__any_sync(0xffffffffu, mx > m_used + GROW)) {
                            // move to the new maximum what has been summed against the old one: O (S(j) follows the product of the
                            // group's last tile, so O is complete), the sum, and this tile's probabilities so far
                            const float m_new = fmaxf(m_used, mx), f = m_new == -INFINITY ? 1.f : exp2f(m_used - m_new);
                            if (begun) scale_columns(tmem_o, HD, f);
                            if (q > 0) scale_packed<FP8>(tmem_s, 16 * q, f);
                            l *= f;
                            sum2[0] = __fmul2_rn(sum2[0], make_float2(f, f));
                            sum2[1] = __fmul2_rn(sum2[1], make_float2(f, f));
                            m_used = m_new;
                        }
                        const float mb = m_used == -INFINITY ? -SHIFT : m_used - SHIFT;
                        const float2 nm2 = make_float2(-mb, -mb);
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 v = make_float2(x[i], x[i + 1]), y = FP8 ? __ffma2_rn(v, sc2, nm2) : __fadd2_rn(v, nm2);
                            x[i] = exp2f(y.x);
                            x[i + 1] = exp2f(y.y);
                        }
                        uint32_t pk[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            sum2[(i >> 1) & 1] = __fadd2_rn(sum2[(i >> 1) & 1], make_float2(x[i], x[i + 1]));
                            pk[i >> 1] = FP8 ? pack_f16(x[i], x[i + 1]) : pack_bf16(x[i], x[i + 1]);
                        }
                        tc::tmem_st16(tmem_s + 16 * q, pk);        // over the scores of columns that this thread has read
                    }
                    l += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
                    tc::tmem_st_wait();
                }
                if (odd_any) {
                    // ---- values that are not finite: rows that see the token get its products here, the others never meet it
                    uint8_t* op = sV + vs * L::VT;
                    if (!tc::mbar_wait(&v_ready[vs], (uint32_t)(j / L::VST) & 1u, abort_flag)) { ok = false; break; }
                    bool have_o = begun;
                    for (int tk = 0; tk < TT && live; ++tk) {
                        if (!(mt.odd[tk >> 5] >> (tk & 31) & 1u)) continue;
                        uint32_t two = 0, pk[16];
                        tc::tmem_ld16(tmem_s + (tk >> 5) * 16, pk);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 16; ++c)
                            if (c == ((tk >> 1) & 15)) two = pk[c];
                        two = tk & 1 ? two >> 16 : two & 0xffffu;
                        const float pv = FP8 ? f16x2_to_float(two).x : __uint_as_float(two << 16);
                        const bool sees_it = seen[tk >> 6] >> (tk & 63) & 1ull;
#pragma unroll 1
                        for (int c = 0; c < HD; c += 16) {
                            uint32_t o[16];
                            tc::tmem_ld16(tmem_o + c, o);
                            tc::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int d = c + i;
                                const uint16_t bits = *reinterpret_cast<const uint16_t*>(op + (d >> 6) * HALF + tk * 128 + ((((d & 63) >> 3) ^ (tk & 7)) << 4) + (d & 7) * 2);
                                const float v = FP8 ? f16x2_to_float(bits).x : __uint_as_float((uint32_t)bits << 16);
                                const float was = have_o ? __uint_as_float(o[i]) : 0.f;
                                o[i] = __float_as_uint(sees_it ? was + pv * v : was);
                            }
                            tc::tmem_st16(tmem_o + c, o);
                        }
                        tc::tmem_st_wait();
                        have_o = true;
                    }
                    if (!exchange(&slow[g], n_slow)) { ok = false; break; }        // the group's rows have read the tokens
                    for (int tk = warp & 3; tk < TT; tk += 4)
                        if ((mt.odd[tk >> 5] >> (tk & 31) & 1u) && lane < HD / 8)
                            *reinterpret_cast<uint4*>(op + (lane >> 3) * HALF + tk * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    tc::fence_proxy_async();
                }
                begun = true;
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&p_ready[g]);
            }
            if (!ok) break;
            // ---- the unit's rows, as far as this part has them: the groups' results together
            row_buf[g * TT + r] = m_used;
            row_buf[(2 + g) * TT + r] = FP8 ? l * 0.0625f : l;
            if (FP8) D = E == OWN ? exp2f(D) : pow2_biased(E) * 9.765625e-4f;     // 2^(E - 127 - 6) and the 2^4 of P
            if (!exchange(&xch, n_x)) { ok = false; break; }
            const int j_last = j0 + len - 1;
            if (!tc::mbar_wait(&pv_done[j_last % L::VST], (uint32_t)(j_last / L::VST) & 1u, abort_flag)) { ok = false; break; }
            tc::tc_fence_after();
            if (live) {
                const bool done = sg.t0 == 0 && sg.t1 == sg.T, mine = R < M;
                const long long slot = 2ll * blockIdx.x + (sg.t0 == 0);
                const float m0 = row_buf[r], m1 = row_buf[TT + r], m = fmaxf(m0, m1), mb = m == -INFINITY ? 0.f : m;
                float f0 = exp2f(m0 - mb), f1 = exp2f(m1 - mb);
                // (a sum without a maximum is zero, or NaN and has to get through)
                const float sum = (m0 == -INFINITY ? row_buf[2 * TT + r] : row_buf[2 * TT + r] * f0) +
                                  (m1 == -INFINITY ? row_buf[3 * TT + r] : row_buf[3 * TT + r] * f1);
                if constexpr (FP8) {
                    f0 *= row_buf[4 * TT + r];
                    f1 *= row_buf[5 * TT + r];
                }
                if (done) {
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    f0 *= inv;
                    f1 *= inv;
                }
                const bool has0 = len > 1 || (j0 & 1) == 0, has1 = len > 1 || (j0 & 1) == 1;       // what a group without a tile left in O is not its
                bf16* dst = p.out + (long long)(c0 + row_i) * p.out_stride + (long long)(sg.h * p.G + row_g) * HD + g * (HD / 2);
                float* part_o = p.part_o + (slot * (HD / 4) + g * (HD / 8)) * TT * 4 + r * 4;      // [HD / 4][rows][4]: a warp's stores are whole lines
#pragma unroll 1
                for (int c = 0; c < HD / 2; c += 16) {
                    uint32_t a[16], b[16];
                    tc::tmem_ld16(tmem_oacc + lane_base + g * (HD / 2) + c, a);
                    tc::tmem_ld16(tmem_oacc + HD + lane_base + g * (HD / 2) + c, b);
                    tc::tmem_ld_wait();
                    if (mine) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            float v[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                v[e] = (has0 ? __uint_as_float(a[i + e]) * f0 : 0.f) + (has1 ? __uint_as_float(b[i + e]) * f1 : 0.f);
                            if (done) *reinterpret_cast<uint2*>(dst + c + i) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
                            else *reinterpret_cast<float4*>(part_o + (long long)((c + i) >> 2) * TT * 4) = make_float4(v[0], v[1], v[2], v[3]);
                        }
                    }
                }
                if (mine && !done && g == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * TT + r) * 2) = make_float2(m, sum);
            }
            tc::tc_fence_before();                     // O is read before the next unit's first products (ordered by their p_ready)
            if (!exchange(&xch, n_x)) { ok = false; break; }
            j0 += len;
        }
        if (!ok && lane == 0) atomicMax(p.status, (int)KB_TIMEOUT_EPI);
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem0, 512);
    }
}

template <bool FP8, int HD>
int run_tile(const TreeParams& p, int grid, cudaStream_t st) {
    static bool flags[64] = {};
    bool* set = kb_device_flag(flags);
    if (!set) return 7;
    if (!*set) {
        if (cudaFuncSetAttribute(tree_tile_kernel<FP8, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<FP8, HD>::SMEM) != cudaSuccess) return 7;
        *set = true;
    }
    return kb_launch_dep(tree_tile_kernel<FP8, HD>, dim3(grid), dim3(THREADS), Lay<FP8, HD>::SMEM, st, p);
}

}  // namespace

int tree::launch_tile(const TreeParams& p, int hd, bool fp8, int grid, cudaStream_t st) {
    if (fp8) return hd == 128 ? run_tile<true, 128>(p, grid, st) : run_tile<true, 64>(p, grid, st);
    return hd == 128 ? run_tile<false, 128>(p, grid, st) : run_tile<false, 64>(p, grid, st);
}
