// Tree attention for many query rows per KV head (drafted tokens times query heads of the group): tiles of 128 rows x 128 cached tokens on
// tcgen05.  The work is cut as in tree_attn_sm100.cu (units of 128 rows, all units' tiles one line, equal parts, merge kernel); here a
// part is walked by one CTA per SM with a role per warp:
//
//   warps 0-7    softmax: two threads per row, 64 token columns each (the row's maximum and sum cross through shared memory)
//   warps 8-11   values: thread t owns token t of the tile.  Query rows -> tensor memory at the start of a unit; what of the tile exists;
//                8-bit pages: factors of the tokens, codes of the values -> f16 operand tile
//   warp 12      MMA issue (the whole warp walks the loop, one elected lane issues)
//   warps 13, 14 TMA of keys and values, a page per lane
//
//   S = Q K^T    A = queries in tensor memory, B = key tile in shared memory (K-major)
//                bf16 pages: kind::f16.  8-bit pages: kind::f8f6f4 on the codes as they lie in the cache; a query row, a power of two
//                taken out, is the sum of two e4m3 numbers, hi + lo, which together hold bf16's eight bits (down to 2^-10 of the row's
//                largest; below that the error is at most 2^-18 of the largest) - two products at twice the rate of one in 16 bits.
//   softmax      in fp32, lazy rescaling (O moves only when a row's maximum grows by more than 2^8); P back to tensor memory in 16 bits
//   O += P V     A = P in tensor memory, B = value tile in shared memory (MN-major).  8-bit pages: P is f16 and carries the token's
//                power of two relative to E, the unit's largest so far, times 2^6 (2^14 with the 2^8 of lazy rescaling), so that it keeps
//                eleven bits down to 2^-20 and is off by at most 2^-31 below; O is in units of 2^(E - 6).
//
// S is double-buffered: the scores of the next tile exist before the softmax of the current one ends.  Query rows are double-buffered by unit.
// Tokens that do not exist are masked in S and zeroed in the value tile (whatever the cache holds there).  Values of drafted tokens that
// are not finite must not meet the zero probabilities of rows that do not see them: such tokens are taken out of the value tile and
// added row by row (never in normal use).  All waits are bounded (status word on timeout).
#include "attn_common.cuh"
#include "tree_attn.cuh"

namespace {

using namespace tree;

constexpr int TT = 128, THREADS = 480;
constexpr int W_VAL = 8, W_MMA = 12, W_K = 13, W_V = 14;
constexpr float GROW = 8.0f;                           // log2 units
constexpr int EMU = 2;                                 // of every 4 pairs of exponentials, this many run on the FMA pipe
constexpr int HALF = TT * 128;                         // 128 tokens x 128 bytes: 16 KB

template <bool FP8, int HD>
struct Lay {
    static constexpr int ROW_BYTES = FP8 ? HD : 2 * HD;
    static constexpr int HALVES = ROW_BYTES > 128 ? 2 : 1, ROWB = ROW_BYTES / HALVES;      // bytes of a staged row
    static constexpr int PIECE = TT * ROWB;            // one half of a staged tile
    static constexpr int KT = HALVES * PIECE;          // a staged tile of keys (or of values)
    static constexpr int VT = HD / 64 * HALF;          // a 16-bit value tile
    // stages of keys, of staged values, of value operand tiles (bf16: the staged tiles themselves)
    static constexpr int KST = FP8 ? 4 : 3, RST = 3, VST = FP8 ? 2 : RST;
    static constexpr int RING = KST * KT + RST * KT + (FP8 ? VST * VT : 0);
    static constexpr int EXPS = FP8 ? RST * 2 * TT : 0;
    static constexpr int FACT = FP8 ? VST * 2 * TT * 4 : 0;
    static constexpr int ROWBUF = 6 * TT * 4;
    static constexpr int SMEM = 1024 + RING + EXPS + FACT + ROWBUF;
};

__device__ __forceinline__ void mma_f8_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], db, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 f16x2_to_float(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// eight bf16 numbers of a query row (rows are 8-byte aligned)
__device__ __forceinline__ uint4 ld_row(const bf16* p) {
    const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + 4);
    return make_uint4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ uint32_t largest(uint32_t two) { return max(two & 0x7fffu, (two >> 16) & 0x7fffu); }

struct TileMeta {                                      // of an operand stage
    uint32_t valid[4], odd[4];                         // bits of the tile's tokens: exist; drafted with values that are not finite
    int E;                                             // biased exponent of the output's unit (8-bit pages)
};

template <bool FP8, int HD>
__global__ void __launch_bounds__(THREADS, 1)
tree_tile_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const TreeParams p) {
    using L = Lay<FP8, HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sK = smem;
    uint8_t* sR = sK + L::KST * L::KT;                                 // staged values
    uint8_t* sV = FP8 ? sR + L::RST * L::KT : sR;                      // value operand tiles
    uint8_t* exps = smem + L::RING;                                    // [RST][2][TT] exponents of keys and values
    float* fact = reinterpret_cast<float*>(exps + L::EXPS);            // [2][2][TT] factors of scores and probabilities
    float* row_buf = reinterpret_cast<float*>(exps + L::EXPS + L::FACT);   // [2 parities][2 halves][TT] maxima, then [2 halves][TT] sums
    __shared__ int uoff[MAX_B + 1];
    __shared__ int wsum[THREADS / 32];
    __shared__ uint64_t k_full[L::KST], k_empty[L::KST], r_full[L::RST], r_empty[L::RST], v_ready[L::VST], pv_done[L::VST], s_full[2], p_ready[2], q_ready[2],
        xch, slow;
    __shared__ uint32_t there[L::RST];                 // bit per page of the staged values: loaded
    __shared__ uint32_t there_k[8];                    // the same of key tile j % 8 (the softmax is less than eight tiles behind the loads)
    __shared__ TileMeta meta[L::VST];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::KST; ++i) { tc::mbar_init(&k_full[i], 1); tc::mbar_init(&k_empty[i], 1); }
        for (int i = 0; i < L::RST; ++i) { tc::mbar_init(&r_full[i], 1); tc::mbar_init(&r_empty[i], 4); }
        for (int i = 0; i < L::VST; ++i) { tc::mbar_init(&v_ready[i], 4); tc::mbar_init(&pv_done[i], 1); }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&s_full[i], 1);
            tc::mbar_init(&p_ready[i], 8);
            tc::mbar_init(&q_ready[i], 4);
        }
        tc::mbar_init(&xch, 8);
        tc::mbar_init(&slow, 8);
        abort_word = 0;
        tc::fence_barrier_init();
        tc::prefetch_tmap(&tmK);
        tc::prefetch_tmap(&tmV);
    }
    if (warp == W_MMA) {
        tc::tmem_alloc(&tmem_slot, 512);
        tc::tmem_relinquish();
    }
    kb_dep_trigger();
    kb_dep_wait();
    tc::tc_fence_before();
    count_tiles<TT, TT, THREADS>(p, uoff, wsum);       // (has the block's barriers)
    tc::tc_fence_after();
    const uint32_t tmem0 = tmem_slot, tmem_oacc = tmem0 + 256, tmem_q = tmem0 + 384;       // S: two times 128 columns; Q: two times 64
    const int2 part = part_of_line(uoff[p.B]);
    const int lo = part.x, n_tiles = part.y - part.x;
    auto segment = [&](int j) { return segment_at<TT, TT>(p, uoff, lo + j, lo + n_tiles); };
    bool ok = true;

    if (n_tiles == 0) {
        // more blocks than tiles
    } else if (warp == W_K || warp == W_V) {
        // ------------------------------------------------------------ TMA: lane l < 8 brings page l of the tile
        const bool isv = warp == W_V;
        Segment sg = segment(0);
        int first = 0;                                 // tile at which sg begins
        int next = -2;                                 // page of the next tile (-2: behind the context)
        auto fetch = [&](int j) {
            if (j >= n_tiles) return;
            if (j - first >= sg.t1 - sg.t0) {
                sg = segment(j);
                first = j;
            }
            const int tok = (sg.t0 + j - first) * TT + lane * PAGE;
            next = lane < 8 && tok < sg.ctx ? p.table[(long long)sg.b * p.max_pages + tok / PAGE] : -2;
        };
        fetch(0);
        for (int j = 0; j < n_tiles; ++j) {
            const int st = isv ? j % L::RST : j % L::KST, use = isv ? j / L::RST : j / L::KST;
            const bool good = next >= 0 && next < p.num_pages;
            if (next != -2 && !good && isv) atomicMax(p.status, (int)KB_BAD_INDEX);
            const long long cell = (long long)next * p.n_kv + sg.h;
            const uint32_t have = __ballot_sync(0xffffffffu, good);
            fetch(j + 1);
            uint64_t* full = isv ? &r_full[st] : &k_full[st];
            if (isv && !FP8) {                         // the stage is the operand tile: free when its product has run
                if (use > 0) ok = tc::mbar_wait(&pv_done[st], (uint32_t)(use - 1) & 1u, abort_flag);
            } else {
                ok = tc::mbar_wait(isv ? &r_empty[st] : &k_empty[st], (uint32_t)(use & 1) ^ 1u, abort_flag);
            }
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            if (lane == 0) {
                if (isv) there[st] = have;
                else there_k[j % 8] = have;
                tc::mbar_expect_tx(full, __popc(have) * (PAGE * L::ROW_BYTES + (FP8 && isv ? 2 * PAGE : 0)));
            }
            __syncwarp();
            if (good) {
                uint8_t* dst = (isv ? sR : sK) + st * L::KT + lane * PAGE * L::ROWB;
#pragma unroll
                for (int h = 0; h < L::HALVES; ++h) tc::tma_load_3d(dst + h * L::PIECE, isv ? &tmV : &tmK, full, 0, (int)(cell * PAGE), h);
                if (FP8 && isv) {
                    uint8_t* e = exps + st * 2 * TT + lane * PAGE;
                    bulk_16(e, p.ke + cell * PAGE, full);
                    bulk_16(e + TT, p.ve + cell * PAGE, full);
                }
            }
        }
        if (!ok && lane == 0) {
            atomicMax(p.status, (int)KB_TIMEOUT_TMA);
            const uint64_t t0 = global_timer_ns();     // copies in flight land before the block can exit
            while (global_timer_ns() - t0 < 2000000ull) {}
        }
    } else if (warp == W_MMA) {
        // ------------------------------------------------------------ products
        const uint32_t id_s = FP8 ? (1u << 4) | (uint32_t)(TT >> 3) << 17 | (uint32_t)(TT >> 4) << 24 : tc::instr_desc_f16(TT, TT, 1, 1, 0, 0);
        const uint32_t id_o = tc::instr_desc_f16(TT, HD, FP8 ? 0 : 1, FP8 ? 0 : 1, 0, 1);
        tc::DescHalves dk = tc::smem_desc_halves(smem_u32(sK), 16, L::ROWB * 8);
        if (L::ROWB == 64) dk.hi = (dk.hi & ~(7u << 29)) | 4u << 29;       // rows of 64 bytes: 64-byte swizzle
        const tc::DescHalves dv = tc::smem_desc_halves(smem_u32(sV), HALF, 1024);
        Segment sg = segment(0);
        int s_left = sg.t1 - sg.t0, s_seg = 0;         // tiles of the segment that S is at; its number
        auto scores = [&](int j) {                     // S(j): waits for its queries and keys
            if (s_left == 0) {
                sg = segment(j);
                s_left = sg.t1 - sg.t0;
                ++s_seg;
            }
            --s_left;
            const int st = j % L::KST;
            if (!tc::mbar_wait(&q_ready[s_seg & 1], (uint32_t)(s_seg >> 1) & 1u, abort_flag)) return false;
            if (!tc::mbar_wait(&k_full[st], (uint32_t)(j / L::KST) & 1u, abort_flag)) return false;
            tc::tc_fence_after();
            const uint32_t b_lo = dk.lo + st * (L::KT >> 4), aq = tmem_q + (s_seg & 1) * 64, d = tmem0 + (j & 1) * 128;
            if (tc::elect_one()) {
                if constexpr (FP8) {
#pragma unroll
                    for (int k = 0; k < HD / 32; ++k) mma_f8_ts(d, aq + 8 * k, b_lo + (k * 32 >> 4), dk.hi, id_s, k != 0);
#pragma unroll
                    for (int k = 0; k < HD / 32; ++k) mma_f8_ts(d, aq + 32 + 8 * k, b_lo + (k * 32 >> 4), dk.hi, id_s, 1u);
                } else {
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k)
                        tc::mma_f16_ts_h(d, aq + 8 * k, b_lo + (((k >> 2) * HALF + (k & 3) * 32) >> 4), dk.hi, id_s, k != 0);
                }
                tc::tc_commit(&s_full[j & 1]);
                tc::tc_commit(&k_empty[st]);
            }
            __syncwarp();
            return true;
        };
        Segment og = sg;
        int o_at = 0, o_len = og.t1 - og.t0;           // tile of the segment that O is at
        ok = scores(0) && (n_tiles < 2 || scores(1));
        for (int j = 0; j < n_tiles && ok; ++j) {
            if (o_at == o_len) {
                og = segment(j);
                o_len = og.t1 - og.t0;
                o_at = 0;
            }
            const int vs = j % L::VST;
            ok = tc::mbar_wait(&v_ready[vs], (uint32_t)(j / L::VST) & 1u, abort_flag) && tc::mbar_wait(&p_ready[j & 1], (uint32_t)(j >> 1) & 1u, abort_flag);
            if (!ok) break;
            tc::tc_fence_after();
            // a first tile overwrites O, unless the softmax warps have begun it (values that are not finite)
            const uint32_t acc = o_at > 0 || (meta[vs].odd[0] | meta[vs].odd[1] | meta[vs].odd[2] | meta[vs].odd[3]) ? 1u : 0u;
            const uint32_t b_lo = dv.lo + vs * (L::VT >> 4), a = tmem0 + (j & 1) * 128;
            if (tc::elect_one()) {
#pragma unroll
                for (int k = 0; k < TT / 16; ++k) tc::mma_f16_ts_h(tmem_oacc, a + 8 * k, b_lo + (k * 2048 >> 4), dv.hi, id_o, k == 0 ? acc : 1u);
                tc::tc_commit(&pv_done[vs]);
            }
            __syncwarp();
            ++o_at;
            if (j + 2 < n_tiles) ok = scores(j + 2);
        }
        if (!ok && lane == 0) atomicMax(p.status, (int)KB_TIMEOUT_MMA);
    } else if (warp >= W_VAL) {
        // ------------------------------------------------------------ values: thread = token of the tile, and = query row
        const int t = threadIdx.x - W_VAL * 32;
        const uint32_t lane_base = (uint32_t)((warp - W_VAL) * 32) << 16;
        auto load_queries = [&](const Segment& sg, int seg) {
            const int R = sg.rb * TT + t;
            const bool live = R < sg.n * p.G;
            const bf16* src = p.q + (long long)((p.cu ? p.cu[sg.b] : sg.b) + (live ? R / p.G : 0)) * p.q_stride + (long long)(sg.h * p.G + (live ? R % p.G : 0)) * HD;
            const uint32_t dst = tmem_q + (seg & 1) * 64 + lane_base;
            if constexpr (FP8) {
                uint32_t big = 0;
#pragma unroll
                for (int i = 0; i < HD / 8; ++i) {
                    const uint4 v = live ? ld_row(src + i * 8) : make_uint4(0u, 0u, 0u, 0u);
                    big = max(big, max(max(largest(v.x), largest(v.y)), max(largest(v.z), largest(v.w))));
                }
                // the largest number comes to [2^7, 2^8); a row that is not finite becomes NaN
                const float inv = big >= 0x7f80u ? __uint_as_float(0x7fc00000u) : pow2_biased(min(254 - (int)(big >> 7) + 7, 254));
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {    // 32 numbers: eight columns of hi, eight of lo
                    uint32_t hi8[8], lo8[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 v = live ? ld_row(src + c * 32 + i * 8) : make_uint4(0u, 0u, 0u, 0u);
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            uint32_t h2[2], l2[2];
#pragma unroll
                            for (int z = 0; z < 2; ++z) {
                                const float a = __uint_as_float(w[2 * e + z] << 16) * inv, b = __uint_as_float(w[2 * e + z] & 0xffff0000u) * inv;
                                h2[z] = e4m3x2(a, b);
                                const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)h2[z], __NV_E4M3)));
                                l2[z] = e4m3x2(a - back.x, b - back.y);
                            }
                            hi8[2 * i + e] = h2[0] | h2[1] << 16;
                            lo8[2 * i + e] = l2[0] | l2[1] << 16;
                        }
                    }
                    tc::tmem_st8(dst + 8 * c, hi8);
                    tc::tmem_st8(dst + 32 + 8 * c, lo8);
                }
            } else {
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 v = live ? ld_row(src + c * 32 + i * 8) : make_uint4(0u, 0u, 0u, 0u);
                        w[4 * i] = v.x;
                        w[4 * i + 1] = v.y;
                        w[4 * i + 2] = v.z;
                        w[4 * i + 3] = v.w;
                    }
                    tc::tmem_st16(dst + 16 * c, w);
                }
            }
            tc::tmem_st_wait();
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&q_ready[seg & 1]);
        };
        Segment sg = segment(0);
        int at = 0, seg = 0, loaded = 0, E = 0;        // tile within the segment, its number; segments whose queries are loaded
        for (int j = 0; j < n_tiles; ++j, ++at) {
            const int vs = j % L::VST, rst = j % L::RST;
            if (at == sg.t1 - sg.t0) {
                sg = segment(j);
                at = 0;
                ++seg;
            }
            // FP8: the operand stage is free when the product two tiles back has run
            const bool ahead = at == 1 && loaded == seg + 1 && j - at + (sg.t1 - sg.t0) < n_tiles;
            if (j >= 2 && (FP8 || loaded <= seg || ahead))
                ok = tc::mbar_wait(&pv_done[(j - 2) % L::VST], (uint32_t)((j - 2) / L::VST) & 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            // queries of this unit, or of the next one once the products of the unit before this one (the buffer's last reader) have run
            if (loaded <= seg) {
                load_queries(sg, seg);
                loaded = seg + 1;
            } else if (ahead) {
                load_queries(segment(j - at + (sg.t1 - sg.t0)), seg + 1);
                loaded = seg + 2;
            }
            ok = tc::mbar_wait(&r_full[rst], (uint32_t)(j / L::RST) & 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            const int base = (sg.t0 + at) * TT, prefix = sg.ctx - sg.n, tok = base + t;
            const uint32_t have = there[rst];
            const bool valid = tok < sg.ctx && (have >> (t / PAGE) & 1u);
            const bool edge = have != 0xffu || base + TT > prefix;
            uint8_t* raw = sR + rst * L::KT;
            uint8_t* op = sV + vs * L::VT;
            uint32_t vword = 0xffffffffu, oword = 0u;
            if (edge) {
                vword = __ballot_sync(0xffffffffu, valid);
                bool bad = false;
                if (valid && tok >= prefix)
                    for (int h = 0; h < L::HALVES; ++h)
                        for (int c = 0; c < L::ROWB / 16; ++c) {
                            const uint4 v = *reinterpret_cast<const uint4*>(raw + h * L::PIECE + t * L::ROWB + c * 16);
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                bad |= FP8 ? __vcmpeq4(w[q] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0u : __vcmpeq2(w[q] & 0x7f807f80u, 0x7f807f80u) != 0u;
                        }
                oword = __ballot_sync(0xffffffffu, bad);
            }
            if constexpr (FP8) {
                // the unit of the output: largest exponent of the values so far (every warp finds it from all 128 tokens)
                const uint8_t* e = exps + rst * 2 * TT;
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int x = e[TT + i * 32 + lane], tk = base + i * 32 + lane;
                    if (x != 255 && (!edge || (tk < sg.ctx && (have >> (2 * i + (lane >> 4)) & 1u)))) top = max(top, (uint32_t)x);
                }
                top = __reduce_max_sync(0xffffffffu, top);
                E = at == 0 ? (int)top : max(E, (int)top);
                const int ek = e[t], ev = e[TT + t], w = min(ev - E, 0) + 6 + 127;
                fact[vs * 2 * TT + t] = pow2_biased(ek);
                fact[vs * 2 * TT + TT + t] = !valid || w <= 0 ? 0.f : ev == 255 ? 1.f : __uint_as_float((uint32_t)w << 23);
                // codes -> f16: a warp takes whole rows, 16 codes per lane, so that loads and stores use all banks
                constexpr int CH = HD / 16, RPW = 32 / CH;     // chunks per row, rows per warp step
                const int c = lane % CH;
#pragma unroll
                for (int i = 0; i < 32 / RPW; ++i) {
                    const int row = (warp - W_VAL) * 32 + i * RPW + lane / CH;
                    const int sw = HD == 128 ? row & 7 : (row >> 1) & 3;
                    uint4 v = *reinterpret_cast<const uint4*>(raw + row * L::ROWB + ((c ^ sw) << 4));
                    if (edge && !(vword >> (row & 31) & 1u)) v = make_uint4(0u, 0u, 0u, 0u);
                    uint4 a, b;
                    codes_to_f16(v.x, a.x, a.y);
                    codes_to_f16(v.y, a.z, a.w);
                    codes_to_f16(v.z, b.x, b.y);
                    codes_to_f16(v.w, b.z, b.w);
                    uint8_t* dst = op + (c >> 2) * HALF + row * 128;
                    const int c0 = (c & 3) * 2, flip = (c >> 2) & 1;       // the two halves of a row share banks: store them in opposite order
                    *reinterpret_cast<uint4*>(dst + (((c0 + flip) ^ (row & 7)) << 4)) = flip ? b : a;
                    *reinterpret_cast<uint4*>(dst + (((c0 + 1 - flip) ^ (row & 7)) << 4)) = flip ? a : b;
                }
            } else if (edge && !valid) {
#pragma unroll
                for (int h = 0; h < L::HALVES; ++h)
                    for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(op + h * HALF + t * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            if (lane == 0) {
                meta[vs].valid[warp - W_VAL] = vword;
                meta[vs].odd[warp - W_VAL] = oword;
                meta[vs].E = E;
            }
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                tc::mbar_arrive(&v_ready[vs]);
                if (FP8) tc::mbar_arrive(&r_empty[rst]);
            }
        }
        if (!ok && lane == 0) atomicMax(p.status, (int)KB_TIMEOUT_TMA);
    } else {
        // ------------------------------------------------------------ softmax: two threads per row
        const int hf = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, tmem_o = tmem_oacc + lane_base;
        uint32_t n_slow = 0, n_x = 0;
        auto exchange = [&](uint64_t* bar, uint32_t& count) {
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar);
            const bool good = tc::mbar_wait(bar, count & 1u, abort_flag);
            ++count;
            return good;
        };
        int j = 0;
        while (j < n_tiles && ok) {
            const Segment sg = segment(j);
            const int M = sg.n * p.G, R = sg.rb * TT + r, c0 = p.cu ? p.cu[sg.b] : sg.b, prefix = sg.ctx - sg.n;
            const bool live = sg.rb * TT + (warp & 3) * 32 < M;            // the warp has rows
            const int row_i = min(R, M - 1) / p.G;
            float scale = p.scale_log2;
            if constexpr (FP8) {                       // the power of two that load_queries took out of this row
                if (live) {
                    const bf16* src = p.q + (long long)(c0 + row_i) * p.q_stride + (long long)(sg.h * p.G + min(R, M - 1) % p.G) * HD + hf * (HD / 2);
                    uint32_t big = 0;
#pragma unroll
                    for (int i = 0; i < HD / 8; ++i) {
                        const uint2 v = *reinterpret_cast<const uint2*>(src + i * 4);
                        big = max(big, max(max(v.x & 0x7fffu, (v.x >> 16) & 0x7fffu), max(v.y & 0x7fffu, (v.y >> 16) & 0x7fffu)));
                    }
                    row_buf[(4 + hf) * TT + r] = __uint_as_float(big);
                }
                if (!exchange(&xch, n_x)) { ok = false; break; }
                const uint32_t big = max(__float_as_uint(row_buf[4 * TT + r]), __float_as_uint(row_buf[5 * TT + r]));
                // 1 / inv of load_queries; exact, both are powers of two
                scale *= pow2_biased(254 - min(254 - (int)(big >> 7) + 7, 254));
                if (!exchange(&xch, n_x)) { ok = false; break; }           // both have read before the sums are written there
            }
            float m_used = -INFINITY, l = 0.f;
            int E = 0;
            for (int at = 0; at < sg.t1 - sg.t0; ++at, ++j) {
                const int vs = j % L::VST, base = (sg.t0 + at) * TT;
                const uint32_t tmem_s = tmem0 + (j & 1) * 128 + lane_base;
                if (!tc::mbar_wait(&s_full[j & 1], (uint32_t)(j >> 1) & 1u, abort_flag)) { ok = false; break; }
                tc::tc_fence_after();
                // tiles with drafted tokens, with the end of the context, or with pages that are not there
                const bool edge = base + TT > prefix || there_k[j % 8] != 0xffu;
                if ((FP8 || edge) && !tc::mbar_wait(&v_ready[vs], (uint32_t)(j / L::VST) & 1u, abort_flag)) { ok = false; break; }
                const TileMeta& mt = meta[vs];
                uint32_t odd_any = 0;
                unsigned long long seen = ~0ull;
                float s[64];
                float mx = -INFINITY;
                if (edge) odd_any = mt.odd[0] | mt.odd[1] | mt.odd[2] | mt.odd[3];
                if (live) {
                    tc::tmem_ld32(tmem_s + hf * 64, reinterpret_cast<uint32_t*>(s));
                    tc::tmem_ld32(tmem_s + hf * 64 + 32, reinterpret_cast<uint32_t*>(s + 32));
                    tc::tmem_ld_wait();
                    if constexpr (FP8) {
                        const float* kf = fact + vs * 2 * TT + hf * 64;
#pragma unroll
                        for (int c = 0; c < 64; c += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(kf + c);
                            const float2 a = __fmul2_rn(make_float2(s[c], s[c + 1]), make_float2(f.x, f.y));
                            const float2 b = __fmul2_rn(make_float2(s[c + 2], s[c + 3]), make_float2(f.z, f.w));
                            s[c] = a.x;
                            s[c + 1] = a.y;
                            s[c + 2] = b.x;
                            s[c + 3] = b.y;
                        }
                    }
                    if (edge) {
                        seen = sees(p, c0, row_i, base + hf * 64 - prefix) &
                               ((unsigned long long)mt.valid[2 * hf] | (unsigned long long)mt.valid[2 * hf + 1] << 32);
#pragma unroll
                        for (int c = 0; c < 64; ++c) s[c] = (uint32_t)(seen >> c) & 1u ? s[c] : -INFINITY;
                    }
                    float mx8[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) mx8[i] = fmaxf(s[2 * i], s[2 * i + 1]);
#pragma unroll
                    for (int c = 16; c < 64; c += 16) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) mx8[i] = attn::fmax3(mx8[i], s[c + 2 * i], s[c + 2 * i + 1]);
                    }
                    mx = attn::fmax3(attn::fmax3(mx8[0], mx8[1], mx8[2]), attn::fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]));
                    row_buf[((j & 1) * 2 + hf) * TT + r] = mx;
                }
                // (also orders "both halves have read their scores" before either writes P over them)
                if (!exchange(&xch, n_x)) { ok = false; break; }
                if (live) {
                    const int E_new = FP8 ? mt.E : 0;
                    mx = fmaxf(mx, row_buf[((j & 1) * 2 + (hf ^ 1)) * TT + r]) * scale;
                    const bool grow = mx > m_used + GROW;
                    if (at == 0) {
                        m_used = mx;
                        E = E_new;
                    } else if (__any_sync(0xffffffffu, grow) || (FP8 && E_new != E)) {
                        if (!tc::mbar_wait(&pv_done[(j - 1) % L::VST], (uint32_t)((j - 1) / L::VST) & 1u, abort_flag)) { ok = false; break; }
                        tc::tc_fence_after();
                        const float m_new = fmaxf(m_used, mx);
                        const float f = m_new == -INFINITY ? 1.f : exp2f(m_used - m_new);
                        const float fo = FP8 ? f * exp2f((float)(E - E_new)) : f;
#pragma unroll 1
                        for (int c = 0; c < HD / 2; c += 16) {
                            uint32_t o[16];
                            tc::tmem_ld16(tmem_o + hf * (HD / 2) + c, o);
                            tc::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fo);
                            tc::tmem_st16(tmem_o + hf * (HD / 2) + c, o);
                        }
                        tc::tmem_st_wait();
                        l *= f;
                        m_used = m_new;
                        E = E_new;
                    }
                    const float mb = m_used == -INFINITY ? 0.f : m_used;
                    const float2 sc2 = make_float2(scale, scale), nm2 = make_float2(-mb, -mb);
                    if (edge) {                                // exponentials of -infinity have to be zero
#pragma unroll
                        for (int c = 0; c < 64; c += 2) {
                            const float2 x = __ffma2_rn(make_float2(s[c], s[c + 1]), sc2, nm2);
                            s[c] = exp2f(x.x);
                            s[c + 1] = exp2f(x.y);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 64; c += 2) {
                            const float2 e = attn::exp2_pair<EMU>(__ffma2_rn(make_float2(s[c], s[c + 1]), sc2, nm2), c >> 1);
                            s[c] = e.x;
                            s[c + 1] = e.y;
                        }
                    }
                    float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    const float* wf = fact + vs * 2 * TT + TT + hf * 64;
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4) {
                        uint32_t pk[8];
#pragma unroll
                        for (int c = q4 * 16; c < q4 * 16 + 16; c += 4) {
                            float2 a = make_float2(s[c], s[c + 1]), b = make_float2(s[c + 2], s[c + 3]);
                            sum2[0] = __fadd2_rn(sum2[0], a);
                            sum2[1] = __fadd2_rn(sum2[1], b);
                            if constexpr (FP8) {
                                const float4 w = *reinterpret_cast<const float4*>(wf + c);
                                a = __fmul2_rn(a, make_float2(w.x, w.y));
                                b = __fmul2_rn(b, make_float2(w.z, w.w));
                                s[c] = a.x;                    // (kept for the pass below)
                                s[c + 1] = a.y;
                                s[c + 2] = b.x;
                                s[c + 3] = b.y;
                            }
                            pk[(c >> 1) & 7] = FP8 ? pack_f16(a.x, a.y) : pack_bf16(a.x, a.y);
                            pk[((c >> 1) & 7) + 1] = FP8 ? pack_f16(b.x, b.y) : pack_bf16(b.x, b.y);
                        }
                        tc::tmem_st8(tmem_s + hf * 32 + q4 * 8, pk);
                    }
                    l += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
                    tc::tmem_st_wait();
                }
                if (odd_any) {
                    // ---- values that are not finite: rows that see the token get its products here, the others never meet it
                    uint8_t* op = sV + vs * L::VT;
                    if (live && at > 0 && !tc::mbar_wait(&pv_done[(j - 1) % L::VST], (uint32_t)((j - 1) / L::VST) & 1u, abort_flag)) { ok = false; break; }
                    tc::tc_fence_after();
                    bool begun = at > 0;
                    for (int tk = 0; tk < TT; ++tk) {
                        if (!(mt.odd[tk >> 5] >> (tk & 31) & 1u)) continue;
                        if (live && hf == tk >> 6) {
                            float mine = 0.f;
#pragma unroll
                            for (int c = 0; c < 64; ++c)
                                if (c == (tk & 63)) mine = s[c];
                            row_buf[4 * TT + r] = seen >> (tk & 63) & 1ull ? mine : -1.f;
                        }
                        if (!exchange(&slow, n_slow)) { ok = false; break; }
                        if (live) {
                            const float pv = row_buf[4 * TT + r];
#pragma unroll 1
                            for (int c = 0; c < HD / 2; c += 16) {
                                uint32_t o[16];
                                tc::tmem_ld16(tmem_o + hf * (HD / 2) + c, o);
                                tc::tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    const int d = hf * (HD / 2) + c + i;
                                    const uint16_t bits = *reinterpret_cast<const uint16_t*>(op + (d >> 6) * HALF + tk * 128 + ((((d & 63) >> 3) ^ (tk & 7)) << 4) + (d & 7) * 2);
                                    const float v = FP8 ? f16x2_to_float(bits).x : __uint_as_float((uint32_t)bits << 16);
                                    const float was = begun ? __uint_as_float(o[i]) : 0.f;
                                    o[i] = __float_as_uint(pv < 0.f ? was : was + pv * v);
                                }
                                tc::tmem_st16(tmem_o + hf * (HD / 2) + c, o);
                            }
                            tc::tmem_st_wait();
                        }
                        begun = true;
                        if (!exchange(&slow, n_slow)) { ok = false; break; }
                        if (warp == 0 && lane < HD / 8) *reinterpret_cast<uint4*>(op + (lane >> 3) * HALF + tk * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    if (!ok) break;
                    tc::fence_proxy_async();
                }
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&p_ready[j & 1]);
            }
            if (!ok) break;
            // ---- the unit's rows, as far as this part has them
            row_buf[(4 + hf) * TT + r] = l;
            if (!exchange(&xch, n_x)) { ok = false; break; }
            l += row_buf[(4 + (hf ^ 1)) * TT + r];
            if (!tc::mbar_wait(&pv_done[(j - 1) % L::VST], (uint32_t)((j - 1) / L::VST) & 1u, abort_flag)) { ok = false; break; }
            tc::tc_fence_after();
            if (live) {
                const bool done = sg.t0 == 0 && sg.t1 == sg.T, mine = R < M;
                const long long slot = 2ll * blockIdx.x + (sg.t0 == 0);
                float unit = 1.f;
                if constexpr (FP8) unit = pow2_biased(E) * 0.015625f;      // 2^(E - 127 - 6)
                if (done) unit *= l == 0.f ? 0.f : 1.f / l;
                bf16* dst = p.out + (long long)(c0 + row_i) * p.out_stride + (long long)(sg.h * p.G + min(R, M - 1) % p.G) * HD + hf * (HD / 2);
                float* part_o = p.part_o + (slot * TT + r) * HD + hf * (HD / 2);
#pragma unroll 1
                for (int c = 0; c < HD / 2; c += 32) {
                    uint32_t o[32];
                    tc::tmem_ld32(tmem_o + hf * (HD / 2) + c, o);
                    tc::tmem_ld_wait();
                    if (mine) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            float v[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(o[i + e]) * unit;
                            if (done) *reinterpret_cast<uint2*>(dst + c + i) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
                            else *reinterpret_cast<float4*>(part_o + c + i) = make_float4(v[0], v[1], v[2], v[3]);
                        }
                    }
                }
                if (mine && !done && hf == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * TT + r) * 2) = make_float2(m_used, l);
            }
            tc::tc_fence_before();                     // O is read before the next unit's first product (ordered by its p_ready)
            if (!exchange(&xch, n_x)) { ok = false; break; }               // and the sums before the next unit writes there
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
int run_tile(const CUtensorMap& tmK, const CUtensorMap& tmV, const TreeParams& p, int grid, cudaStream_t st) {
    static bool flags[64] = {};
    bool* set = kb_device_flag(flags);
    if (!set) return 7;
    if (!*set) {
        if (cudaFuncSetAttribute(tree_tile_kernel<FP8, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<FP8, HD>::SMEM) != cudaSuccess) return 7;
        *set = true;
    }
    return kb_launch_dep(tree_tile_kernel<FP8, HD>, dim3(grid), dim3(THREADS), Lay<FP8, HD>::SMEM, st, tmK, tmV, p);
}

}  // namespace

int tree::launch_tile(const CUtensorMap& tmK, const CUtensorMap& tmV, const TreeParams& p, int hd, bool fp8, int grid, cudaStream_t st) {
    if (fp8) return hd == 128 ? run_tile<true, 128>(tmK, tmV, p, grid, st) : run_tile<true, 64>(tmK, tmV, p, grid, st);
    return hd == 128 ? run_tile<false, 128>(tmK, tmV, p, grid, st) : run_tile<false, 64>(tmK, tmV, p, grid, st);
}
