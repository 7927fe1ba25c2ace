// Attention of drafted tokens over the paged cache for heads of 64 and 128 in bf16, pages in bf16 or 8 bits (cache_fp8.cu).  What a row
// sees is defined in tree_attn.cu.
//
// What bounds it.  A cached row is used by the (drafted token, query head) rows of its KV head only - 1 to a few hundred - so the
// cache's bytes bound the call, and above ~100 rows the tensor cores do.  Each (sequence, KV head) has its n * G query rows as the
// M side of `mma.sync.m16n8k16` tiles (ROWS = 16 or 32 of them per unit of work), cached tokens are the N side of the score product and
// the K side of the output product; probabilities go from accumulators to operands in registers.
//
// Work.  A unit is (sequence, KV head, block of ROWS rows); its tiles are TILE tokens of the context.  All units' tiles form one line
// that is cut into equal parts, one per CTA, so that ragged contexts and one long context load the GPU alike.  A CTA walks its part:
// a unit that lies inside it is finished there, the others leave partial results (unnormalised output, maximum, sum per row)
// that the merge kernel puts together.  A CTA has at most two such partial units: the one it enters with (slot 0) and the one it leaves with (slot 1).
//
// Inside a CTA the four warps share the rows and split the tokens: warp w has tokens w * IT .. of every tile, in a ring of its own that
// TMA fills page by page (128- or 64-byte swizzle), so nothing in the loop waits for another warp; every cached number is
// converted once per CTA.  The warps' results meet in shared memory at the end of a unit.
//
// 8-bit pages.  Codes become f16 (exact) on the way to the tensor cores.  Keys: the score's accumulator is scaled by the token's power of two.
// Values: the probability is scaled by the token's power of two relative to E, the largest seen so far by the warp, times 2^14, and
// rounded to f16; the output is kept in units of 2^(E - 14).  So a probability keeps f16's eleven bits down to 2^-28 of the largest.
// Queries become f16 with a power of two per row taken out (exact down to 2^-24 of the row's largest).
// bf16 pages: queries as they are, probabilities rounded to bf16 (2^-9 relative, like the other decode kernels).
// Scores, maxima, sums and outputs are fp32.
#include "tree_attn.cuh"

namespace {

using namespace tree;

constexpr int WARPS = 4, THREADS = WARPS * 32;

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool F16>
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A page's rows of one KV head, seen as [halves][16 rows][at most 128 bytes]: bf16 heads of 128 have two halves.
__device__ __forceinline__ void tma_page(void* dst, const CUtensorMap* m, uint64_t* bar, int row) { tc::tma_load_3d(dst, m, bar, 0, row, 0); }
template <bool FP8, int HD, int MI>
struct Cfg {
    static constexpr int ROWS = 16 * MI;
    static constexpr int IT = FP8 ? 32 : 16;           // tokens of a warp's step
    static constexpr int PAGES = IT / PAGE;
    static constexpr int TILE = WARPS * IT;
    static constexpr int ROW_BYTES = FP8 ? HD : 2 * HD;
    static constexpr int PAGE_BYTES = PAGE * ROW_BYTES;
    static constexpr int STAGE = 2 * PAGES * PAGE_BYTES;               // keys, then values
    static constexpr int NST = HD == 128 ? 2 : 4;
    static constexpr int OPAD = FP8 ? 16 : 8;
    static constexpr int OROW = HD + OPAD;
    static constexpr int RING = WARPS * NST * STAGE;
    static constexpr int OBUF = 2 * ROWS * OROW * 4;
    static constexpr int EXPS = FP8 ? WARPS * NST * 2 * IT : 0;        // exponents of a stage: keys, then values
    static constexpr int FACT = FP8 ? WARPS * 2 * IT * 4 : 0;          // the step's factors as fp32
    static constexpr int SMEM = 1024 + RING + OBUF + EXPS + FACT;
};

template <bool FP8, int HD, int MI>
__global__ void __launch_bounds__(THREADS, 2)
tree_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const TreeParams p) {
    using C = Cfg<FP8, HD, MI>;
    constexpr int IT = C::IT, NT = IT / 8, KS = HD / 16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring_all = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* obuf = reinterpret_cast<float*>(ring_all + C::RING);
    uint8_t* exps_all = ring_all + C::RING + C::OBUF;
    float* fact_all = reinterpret_cast<float*>(exps_all + C::EXPS);
    __shared__ int uoff[MAX_B + 1];
    __shared__ int wsum[WARPS];
    __shared__ uint64_t full[WARPS][C::NST];
    __shared__ uint32_t there[WARPS][C::NST];          // bit per page of a stage: loaded
    __shared__ float wm[2][WARPS][C::ROWS], wl[2][WARPS][C::ROWS];
    __shared__ int we[2][WARPS];
    __shared__ int abort_flag;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, qd = lane & 3;
    if (threadIdx.x == 0) {
        for (int w = 0; w < WARPS; ++w)
            for (int s = 0; s < C::NST; ++s) tc::mbar_init(&full[w][s], 1);
        abort_flag = 0;
        tc::fence_barrier_init();
        tc::prefetch_tmap(&tmK);
        tc::prefetch_tmap(&tmV);
    }
    kb_dep_trigger();
    kb_dep_wait();
    count_tiles<C::ROWS, C::TILE, THREADS>(p, uoff, wsum);
    const int2 part = part_of_line(uoff[p.B]);
    const int lo = part.x, hi = part.y;
    if (lo >= hi) return;
    auto segment = [&](int x) { return segment_at<C::ROWS, C::TILE>(p, uoff, x, hi); };

    // ---- producer side of this warp's ring: item k is this warp's step of tile lo + k
    uint8_t* ring = ring_all + (size_t)warp * C::NST * C::STAGE;
    uint8_t* exps = exps_all + warp * C::NST * 2 * IT;
    Segment ps = segment(lo);
    int px = lo, pfirst = lo;                          // next tile to issue; tile at which ps begins
    int next_page = -1;                                // lane l < PAGES: page number of the next item (fetched one item ahead)
    auto fetch_page = [&]() {
        if (px >= hi) return;
        if (px - pfirst >= ps.t1 - ps.t0) {
            ps = segment(px);
            pfirst = px;
        }
        const int tok = (ps.t0 + px - pfirst) * C::TILE + warp * IT + lane * PAGE;
        next_page = -2;                                // nothing to load
        if (lane < C::PAGES && tok < ps.ctx) next_page = p.table[(long long)ps.b * p.max_pages + tok / PAGE];
    };
    fetch_page();
    auto issue = [&]() {                               // loads item px, then looks up the page numbers of the one after it
        if (px >= hi) return;
        const int st = (px - lo) % C::NST;
        const bool good = next_page >= 0 && next_page < p.num_pages;
        if (lane < C::PAGES && next_page != -2 && !good && p.status) atomicMax(p.status, (int)KB_BAD_INDEX);
        const uint32_t have = __ballot_sync(0xffffffffu, lane < C::PAGES && good);
        if (lane == 0) {
            there[warp][st] = have;
            tc::mbar_expect_tx(&full[warp][st], __popc(have) * (2 * C::PAGE_BYTES + (FP8 ? 2 * PAGE : 0)));
        }
        __syncwarp();
        if (lane < C::PAGES && good) {
            uint8_t* dst = ring + (size_t)st * C::STAGE + lane * C::PAGE_BYTES;
            const long long cell = (long long)next_page * p.n_kv + ps.h;
            tma_page(dst, &tmK, &full[warp][st], (int)(cell * PAGE));
            tma_page(dst + C::PAGES * C::PAGE_BYTES, &tmV, &full[warp][st], (int)(cell * PAGE));
            if constexpr (FP8) {
                uint8_t* e = exps + st * 2 * IT + lane * PAGE;
                bulk_16(e, p.ke + cell * PAGE, &full[warp][st]);
                bulk_16(e + IT, p.ve + cell * PAGE, &full[warp][st]);
            }
        }
        ++px;
        fetch_page();
    };
    for (int i = 0; i < C::NST; ++i) issue();

    bool ok = true;
    int parity = 0;
    for (int x = lo; x < hi;) {
        const Segment sg = segment(x);
        const int row0 = sg.rb * C::ROWS, M = sg.n * p.G, prefix = sg.ctx - sg.n;
        const int c0 = p.cu ? p.cu[sg.b] : sg.b;
        // ---- the unit's queries as A fragments
        uint32_t qa[MI][KS][4];
        float rs[MI][2];                               // scores of rows r, r + 8 in log2 units per accumulator unit
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
            uint2 raw[2][KS];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int R = row0 + mi * 16 + hf * 8 + r;
                const bf16* src = p.q + (long long)(c0 + R / p.G) * p.q_stride + (long long)(sg.h * p.G + R % p.G) * HD;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    raw[hf][ks] = make_uint2(0u, 0u);
                    if (R < M) {
                        if constexpr (FP8) raw[hf][ks] = *reinterpret_cast<const uint2*>(src + ks * 16 + 4 * qd);
                        else raw[hf][ks] = make_uint2(*reinterpret_cast<const uint32_t*>(src + ks * 16 + 2 * qd),
                                                      *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8 + 2 * qd));
                    }
                }
                rs[mi][hf] = p.scale_log2;
                if constexpr (FP8) {                   // take a power of two out of the row, then f16
                    uint32_t big = 0;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
                        big = max(big, max(max(raw[hf][ks].x & 0x7fffu, (raw[hf][ks].x >> 16) & 0x7fffu),
                                           max(raw[hf][ks].y & 0x7fffu, (raw[hf][ks].y >> 16) & 0x7fffu)));
                    big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                    big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                    const int e = min(max((int)(big >> 7), 1), 253);       // biased exponent of the largest number
                    const float inv = pow2_biased(254 - e);
                    rs[mi][hf] = p.scale_log2 * pow2_biased(e);
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        const uint32_t a = raw[hf][ks].x, b = raw[hf][ks].y;
                        raw[hf][ks].x = pack_f16(__uint_as_float(a << 16) * inv, __uint_as_float(a & 0xffff0000u) * inv);
                        raw[hf][ks].y = pack_f16(__uint_as_float(b << 16) * inv, __uint_as_float(b & 0xffff0000u) * inv);
                    }
                }
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                qa[mi][ks][0] = raw[0][ks].x;
                qa[mi][ks][1] = raw[1][ks].x;
                qa[mi][ks][2] = raw[0][ks].y;
                qa[mi][ks][3] = raw[1][ks].y;
            }
        }
        float o[MI][HD / 8][4], m[MI][2], l[MI][2];
        int E = 0;                                     // biased exponent of the output's unit
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) o[mi][j][0] = o[mi][j][1] = o[mi][j][2] = o[mi][j][3] = 0.f;
            m[mi][0] = m[mi][1] = -INFINITY;
            l[mi][0] = l[mi][1] = 0.f;
        }
        for (int t = sg.t0; t < sg.t1; ++t, ++x) {
            const int k = x - lo, st = k % C::NST;
            if (ok && !tc::mbar_wait(&full[warp][st], (uint32_t)(k / C::NST) & 1u, &abort_flag)) ok = false;
            ok = __shfl_sync(0xffffffffu, (int)ok, 0);
            const int base = t * C::TILE + warp * IT;
            const uint32_t have = there[warp][st];
            if (ok && have) {
                const uint32_t kb = smem_u32(ring + (size_t)st * C::STAGE), vb = kb + C::PAGES * C::PAGE_BYTES;
                uint32_t valid = 0;                    // tokens of the step that exist
#pragma unroll
                for (int i = 0; i < C::PAGES; ++i) valid |= (have >> i & 1u) * (0xffffu << (16 * i));
                if (base + IT > sg.ctx) valid &= 0xffffffffu >> (32 - (sg.ctx - base));
                const bool whole = valid == (IT == 32 ? 0xffffffffu : 0xffffu);
                const bool drafts = base + IT > prefix;
                float* fk = fact_all + warp * 2 * IT;
                float grow = 1.f;                      // factor of the output's change of unit
                if constexpr (FP8) {
                    const uint8_t* e = exps + st * 2 * IT;
                    const int ek = e[lane], ev = e[IT + lane];
                    const bool counts = (valid >> lane & 1u) && ev != 255;
                    const int top = (int)__reduce_max_sync(0xffffffffu, counts ? (unsigned)ev : 0u);
                    if (top > E) {
                        grow = exp2f((float)(E - top));
                        E = top;
                    }
                    fk[lane] = pow2_biased(ek);
                    const int w = min(ev - E, 0) + 14 + 127;
                    fk[IT + lane] = counts ? (w > 0 ? __uint_as_float((uint32_t)w << 23) : 0.f) : 1.f;
                    __syncwarp();
                }
                // ---- scores
                float s[MI][NT][4];
#pragma unroll
                for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                    for (int j = 0; j < NT; ++j) s[mi][j][0] = s[mi][j][1] = s[mi][j][2] = s[mi][j][3] = 0.f;
                if constexpr (FP8) {
                    const int tok = (lane >> 3) * 8 + (lane & 7);          // ldmatrix: matrix lane / 8 = tokens of n tile lane / 8
                    const uint32_t row = kb + tok * HD;
                    const int sw = HD == 128 ? tok & 7 : (tok >> 1) & 3;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        uint32_t c[4];
                        ldsm_x4(row + ((ks ^ sw) << 4), c);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t b0, b1;
                            codes_to_f16(c[j], b0, b1);
#pragma unroll
                            for (int mi = 0; mi < MI; ++mi) mma<true>(s[mi][j], qa[mi][ks], b0, b1);
                        }
                    }
                } else {
                    const int tok = (lane & 7) + (lane >> 4) * 8, sub = (lane >> 3) & 1;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        const int ch = ks * 2 + sub;
                        uint32_t b[4];
                        ldsm_x4(kb + (ch >> 3) * 2048 + tok * 128 + (((ch & 7) ^ (tok & 7)) << 4), b);
#pragma unroll
                        for (int mi = 0; mi < MI; ++mi) {
                            mma<false>(s[mi][0], qa[mi][ks], b[0], b[1]);
                            mma<false>(s[mi][1], qa[mi][ks], b[2], b[3]);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float2 f = make_float2(1.f, 1.f);
                    if constexpr (FP8) f = *reinterpret_cast<const float2*>(fk + 8 * j + 2 * qd);
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi) {
                        s[mi][j][0] *= f.x * rs[mi][0];
                        s[mi][j][1] *= f.y * rs[mi][0];
                        s[mi][j][2] *= f.x * rs[mi][1];
                        s[mi][j][3] *= f.y * rs[mi][1];
                    }
                }
                // ---- what is not seen: places that hold no token, and drafted tokens the row's mask does not name
                uint32_t odd = 0;                      // drafted tokens whose values are not finite: kept out of the product
                unsigned long long seen[MI][2];        // bit t: the row sees token t of the step (only where something is hidden)
                if (!whole || drafts) {
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            const int i = min((row0 + mi * 16 + hf * 8 + r) / p.G, sg.n - 1);
                            seen[mi][hf] = sees(p, c0, i, base - prefix) & valid;
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                const uint32_t two = (uint32_t)(seen[mi][hf] >> (8 * j + 2 * qd)) & 3u;
                                if (!(two & 1u)) s[mi][j][2 * hf] = -INFINITY;
                                if (!(two & 2u)) s[mi][j][2 * hf + 1] = -INFINITY;
                            }
                        }
                    if (drafts) {
                        bool bad = false;
                        if (lane < IT && (valid >> lane & 1u) && base + lane >= prefix) {
                            const uint8_t* row = ring + (size_t)st * C::STAGE + C::PAGES * C::PAGE_BYTES + (lane / PAGE) * C::PAGE_BYTES;
                            const int tr = lane % PAGE;
                            for (int c = 0; c < C::ROW_BYTES / 16; ++c) {
                                const uint4 v = *reinterpret_cast<const uint4*>(FP8 ? row + tr * HD + c * 16 : row + (c >> 3) * 2048 + tr * 128 + (c & 7) * 16);
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int q = 0; q < 4; ++q)
                                    bad |= FP8 ? __vcmpeq4(w[q] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0u : __vcmpeq2(w[q] & 0x7f807f80u, 0x7f807f80u) != 0u;
                            }
                        }
                        odd = __ballot_sync(0xffffffffu, bad);
                    }
                }
                // ---- online softmax
                uint32_t pa[MI][IT / 16][4];
                bool still = true;
                float f[MI][2];
#pragma unroll
                for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        float mx = -INFINITY;
#pragma unroll
                        for (int j = 0; j < NT; ++j) mx = fmaxf(mx, fmaxf(s[mi][j][2 * hf], s[mi][j][2 * hf + 1]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const float mn = fmaxf(m[mi][hf], mx), at = mn == -INFINITY ? 0.f : mn;
                        const float g = exp2f(m[mi][hf] - at);
                        m[mi][hf] = mn;
                        float sum = 0.f;
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            s[mi][j][2 * hf] = exp2f(s[mi][j][2 * hf] - at);
                            s[mi][j][2 * hf + 1] = exp2f(s[mi][j][2 * hf + 1] - at);
                            sum += s[mi][j][2 * hf] + s[mi][j][2 * hf + 1];
                        }
                        l[mi][hf] = l[mi][hf] * g + sum;
                        f[mi][hf] = g * grow;
                        still = still && f[mi][hf] == 1.f;
                    }
                if (!__all_sync(0xffffffffu, still)) {
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                        for (int j = 0; j < HD / 8; ++j) {
                            o[mi][j][0] *= f[mi][0];
                            o[mi][j][1] *= f[mi][0];
                            o[mi][j][2] *= f[mi][1];
                            o[mi][j][3] *= f[mi][1];
                        }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if constexpr (FP8) {
                        const float2 w = *reinterpret_cast<const float2*>(fk + IT + 8 * j + 2 * qd);
#pragma unroll
                        for (int mi = 0; mi < MI; ++mi) {
                            s[mi][j][0] *= w.x;
                            s[mi][j][1] *= w.y;
                            s[mi][j][2] *= w.x;
                            s[mi][j][3] *= w.y;
                        }
                    }
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf)
                            pa[mi][j >> 1][(j & 1) * 2 + hf] = FP8 ? pack_f16(s[mi][j][2 * hf], s[mi][j][2 * hf + 1])
                                                                   : pack_bf16(s[mi][j][2 * hf], s[mi][j][2 * hf + 1]);
                }
                // ---- output
                const uint32_t use = valid & ~odd;
                const bool cut = !whole || odd;
                const int vtok = (lane & 7) + ((lane >> 3) & 1) * 8, vsub = lane >> 4;
#pragma unroll
                for (int kk = 0; kk < IT / 16; ++kk) {
                    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;     // tokens 2 qd, 2 qd + 1 (+ 8) of the page, 16 bits each
                    if (cut) {
                        const uint32_t a = use >> (16 * kk + 2 * qd), z = use >> (16 * kk + 8 + 2 * qd);
                        keep0 = (a & 1u ? 0xffffu : 0u) | (a & 2u ? 0xffff0000u : 0u);
                        keep1 = (z & 1u ? 0xffffu : 0u) | (z & 2u ? 0xffff0000u : 0u);
                    }
                    if constexpr (FP8) {
                        const int tok = kk * 16 + vtok;
                        const uint32_t row = vb + tok * HD;
                        const int sw = HD == 128 ? tok & 7 : (tok >> 1) & 3;
#pragma unroll
                        for (int c = 0; c < HD / 16; c += 2) {
                            uint32_t v[4];
                            ldsm_x4_t(row + (((c + vsub) ^ sw) << 4), v);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                uint32_t e0, o0, e1, o1;                   // even and odd head dimensions of the chunk
                                codes_to_f16(__byte_perm(v[2 * i] & keep0, 0, 0x3120), e0, o0);
                                codes_to_f16(__byte_perm(v[2 * i + 1] & keep1, 0, 0x3120), e1, o1);
#pragma unroll
                                for (int mi = 0; mi < MI; ++mi) {
                                    mma<true>(o[mi][2 * (c + i)], pa[mi][kk], e0, e1);
                                    mma<true>(o[mi][2 * (c + i) + 1], pa[mi][kk], o0, o1);
                                }
                            }
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < HD / 16; ++j) {
                            const int ch = j * 2 + vsub;
                            uint32_t v[4];
                            ldsm_x4_t(vb + (ch >> 3) * 2048 + vtok * 128 + (((ch & 7) ^ (vtok & 7)) << 4), v);
#pragma unroll
                            for (int mi = 0; mi < MI; ++mi) {
                                mma<false>(o[mi][2 * j], pa[mi][kk], v[0] & keep0, v[1] & keep1);
                                mma<false>(o[mi][2 * j + 1], pa[mi][kk], v[2] & keep0, v[3] & keep1);
                            }
                        }
                    }
                }
                for (uint32_t left = odd; left; left &= left - 1u) {       // rare: rows that see such a token get its products one by one
                    const int tk = __ffs(left) - 1, src = (lane & ~3) | ((tk & 7) >> 1);
                    const uint8_t* row = ring + (size_t)st * C::STAGE + C::PAGES * C::PAGE_BYTES + (tk / PAGE) * C::PAGE_BYTES;
                    const int tr = tk % PAGE;
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            float mine = 0.f;
#pragma unroll
                            for (int j = 0; j < NT; ++j)
                                if (j == tk >> 3) mine = tk & 1 ? s[mi][j][2 * hf + 1] : s[mi][j][2 * hf];
                            const float pv = __shfl_sync(0xffffffffu, mine, src);
                            if (!(seen[mi][hf] >> tk & 1ull)) continue;
#pragma unroll
                            for (int j = 0; j < HD / 8; ++j)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    float v;
                                    if constexpr (FP8) {
                                        const int d = (j >> 1) * 16 + 4 * qd + 2 * e + (j & 1), c = d >> 4;
                                        const int sw = HD == 128 ? tr & 7 : (tr >> 1) & 3;
                                        v = __half2float(__half(__nv_cvt_fp8_to_halfraw(row[tr * HD + ((c ^ sw) << 4) + (d & 15)], __NV_E4M3)));
                                    } else {
                                        const int d = 8 * j + 2 * qd + e, c = d >> 3;
                                        v = __bfloat162float(*reinterpret_cast<const bf16*>(row + (c >> 3) * 2048 + tr * 128 + (((c & 7) ^ (tr & 7)) << 4) + (d & 7) * 2));
                                    }
                                    o[mi][j][2 * hf + e] += pv * v;
                                }
                        }
                }
            }
            __syncwarp();                              // every lane has read the stage
            if (ok) {
                tc::fence_proxy_async();
                issue();
            }
        }
        // ---- the warps' results meet
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                l[mi][hf] += __shfl_xor_sync(0xffffffffu, l[mi][hf], 1);
                l[mi][hf] += __shfl_xor_sync(0xffffffffu, l[mi][hf], 2);
                if (qd == 0) {
                    wm[parity][warp][mi * 16 + hf * 8 + r] = m[mi][hf];
                    wl[parity][warp][mi * 16 + hf * 8 + r] = l[mi][hf];
                }
            }
        if (lane == 0) we[parity][warp] = E;
        __syncthreads();
        const float unit = FP8 ? pow2_biased(E) * 6.103515625e-05f : 1.f;              // 2^(E - 127 - 14)
        float* buf = obuf + (warp & 1) * C::ROWS * C::OROW;
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {
            if ((warp >> 1) == turn) {
#pragma unroll
                for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const int row = mi * 16 + hf * 8 + r;
                        float top = wm[parity][0][row];
#pragma unroll
                        for (int w = 1; w < WARPS; ++w) top = fmaxf(top, wm[parity][w][row]);
                        const float g = m[mi][hf] == -INFINITY ? 0.f : exp2f(m[mi][hf] - top) * unit;
                        const bool none = m[mi][hf] == -INFINITY && l[mi][hf] == 0.f;   // (a NaN sum has to get through)
                        float* dst = buf + row * C::OROW;
#pragma unroll
                        for (int j = 0; j < HD / 8; ++j) {
                            const int d0 = FP8 ? (j >> 1) * 16 + 4 * qd + (j & 1) : 8 * j + 2 * qd, d1 = d0 + (FP8 ? 2 : 1);
                            const float a = none ? 0.f : o[mi][j][2 * hf] * g, z = none ? 0.f : o[mi][j][2 * hf + 1] * g;
                            if (turn == 0) {
                                dst[d0] = a;
                                dst[d1] = z;
                            } else {
                                dst[d0] += a;
                                dst[d1] += z;
                            }
                        }
                    }
            }
            __syncthreads();
        }
        const bool done = sg.t0 == 0 && sg.t1 == sg.T;
        const long long slot = 2ll * blockIdx.x + (sg.t0 == 0);
        for (int i = threadIdx.x; i < C::ROWS * (HD / 4); i += THREADS) {
            const int row = i % C::ROWS, d = i / C::ROWS * 4, R = row0 + row;
            if (R >= M) continue;
            const float4 a = *reinterpret_cast<const float4*>(obuf + row * C::OROW + d);
            const float4 z = *reinterpret_cast<const float4*>(obuf + (C::ROWS + row) * C::OROW + d);
            float4 v = make_float4(a.x + z.x, a.y + z.y, a.z + z.z, a.w + z.w);
            float top = wm[parity][0][row], sum = 0.f;
#pragma unroll
            for (int w = 1; w < WARPS; ++w) top = fmaxf(top, wm[parity][w][row]);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float mw = wm[parity][w][row], lw = wl[parity][w][row];
                sum += mw == -INFINITY ? lw : lw * exp2f(mw - top);          // lw is 0 or NaN where there is no maximum
            }
            if (done) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                bf16* dst = p.out + (long long)(c0 + R / p.G) * p.out_stride + (long long)(sg.h * p.G + R % p.G) * HD + d;
                *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
            } else {
                *reinterpret_cast<float4*>(p.part_o + ((slot * (HD / 4) + d / 4) * C::ROWS + row) * 4) = v;
                if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * C::ROWS + row) * 2) = make_float2(top, sum);
            }
        }
        parity ^= 1;
    }
    if (!ok) {
        // a copy did not arrive in time: report, and let copies in flight land before the shared memory goes
        if (lane == 0) {
            atomicMax(p.status, (int)KB_TIMEOUT_TMA);
            const uint64_t t0 = global_timer_ns();
            while (global_timer_ns() - t0 < 2000000ull) {}
        }
        __syncwarp();
    }
}

// Puts the parts of a unit together; WPR warps share a row.  Rows of sequences without rows or tokens, and (zero_tail) rows behind the
// last sequence, become zero.
template <int HD, int WPR>
__global__ void __launch_bounds__(256)
tree_merge_kernel(const TreeParams p, int ROWS, int TILE, int grid, int zero_tail) {
    kb_dep_trigger();
    kb_dep_wait();
    constexpr int RPB = 8 / WPR, EPL = HD / 32;        // rows per block; dimensions per lane
    __shared__ float so[WPR > 1 ? 8 : 1][HD], sml[8][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR;
    const long long row = (long long)blockIdx.x * RPB + warp / WPR;
    if (row >= (long long)p.N * p.H) return;           // (with WPR = 8 the whole block)
    const int n = (int)(row / p.H), head = (int)(row % p.H), h = head / p.G;
    int b = n;
    if (p.cu) {
        int a = 0, z = p.B;
        while (z - a > 1) {
            const int mid = (a + z) >> 1;
            if (p.cu[mid] <= n) a = mid; else z = mid;
        }
        b = a;
    }
    const int c0 = b < p.B ? (p.cu ? p.cu[b] : b) : 0, c1 = b < p.B ? (p.cu ? p.cu[b + 1] : b + 1) : 0;
    const bool inside = b < p.B && n >= c0 && n < c1;
    bf16* dst = p.out + (long long)n * p.out_stride + (long long)head * HD + lane * EPL;
    const int2 sp = inside ? span_of(p, b, false) : make_int2(0, 0);
    if (sp.x == 0) {
        if ((inside || zero_tail) && sub == 0)
#pragma unroll
            for (int e = 0; e < EPL; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = 0u;
        return;
    }
    const int Rl = (n - c0) * p.G + head % p.G, rbs = (sp.x * p.G + ROWS - 1) / ROWS, T = (sp.y + TILE - 1) / TILE;
    const long long total = p.uoff[p.B], s0 = p.uoff[b] + (long long)(h * rbs + Rl / ROWS) * T;
    const long long parts = min((long long)grid, total);
    const int first = (int)(((s0 + 1) * parts - 1) / total), last = (int)(((s0 + T) * parts - 1) / total);
    if (first == last) return;                         // finished by its CTA
    const int r = Rl % ROWS;
    float M = -INFINITY, L = 0.f, acc[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
    constexpr int U = 4;                               // parts in flight
    for (int j0 = first + sub; j0 <= last; j0 += WPR * U) {
        float2 ml[U];
        float v[U][EPL];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * WPR;
            ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int e = 0; e < EPL; ++e) v[u][e] = 0.f;
            if (j <= last) {
                const long long at = (2ll * j + (j == first)) * ROWS + r;
                ml[u] = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
#pragma unroll
                for (int e = 0; e < EPL; e += 2) {
                    const int d = lane * EPL + e;
                    *reinterpret_cast<float2*>(&v[u][e]) = *reinterpret_cast<const float2*>(p.part_o + (((2ll * j + (j == first)) * (HD / 4) + d / 4) * ROWS + r) * 4 + d % 4);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float mn = fmaxf(M, ml[u].x), at = mn == -INFINITY ? 0.f : mn, f = exp2f(M - at), g = exp2f(ml[u].x - at);
            M = mn;
            L = L * f + (ml[u].x == -INFINITY ? ml[u].y : ml[u].y * g);
#pragma unroll
            for (int e = 0; e < EPL; ++e) acc[e] = acc[e] * f + v[u][e] * g;
        }
    }
    if constexpr (WPR > 1) {
#pragma unroll
        for (int e = 0; e < EPL; ++e) so[warp][lane * EPL + e] = acc[e];
        if (lane == 0) {
            sml[warp][0] = M;
            sml[warp][1] = L;
        }
        __syncthreads();
        if (sub != 0) return;
        float top = M;
#pragma unroll
        for (int w = 1; w < WPR; ++w) top = fmaxf(top, sml[w][0]);
        const float at = top == -INFINITY ? 0.f : top;
        L = 0.f;
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) {
            const float g = exp2f(sml[w][0] - at);
            L += sml[w][0] == -INFINITY ? sml[w][1] : sml[w][1] * g;
#pragma unroll
            for (int e = 0; e < EPL; ++e) acc[e] += so[w][lane * EPL + e] * g;
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < EPL; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
    static EncodeFn enc = nullptr;
    if (!enc) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
        enc = reinterpret_cast<EncodeFn>(ptr);
    }
    return enc;
}
}  // namespace

int tree::page_map(CUtensorMap* m, const void* base, long long rows, int hd, bool fp8, bool halves_apart) {
    const EncodeFn enc = encoder();
    if (!enc) return 100;
    const int row_bytes = fp8 ? hd : 2 * hd, in = row_bytes > 128 ? 128 : row_bytes, esz = fp8 ? 1 : 2;
    const cuuint64_t dims[3] = {(cuuint64_t)(in / esz), (cuuint64_t)rows, (cuuint64_t)(row_bytes / in)};
    const cuuint64_t strides[2] = {(cuuint64_t)row_bytes, (cuuint64_t)in};
    const cuuint32_t box[3] = {(cuuint32_t)(in / esz), PAGE, halves_apart ? 1u : (cuuint32_t)(row_bytes / in)}, one[3] = {1, 1, 1};
    const CUresult r = enc(m, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box,
                           one, CU_TENSOR_MAP_INTERLEAVE_NONE, in == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 200 + (int)r;
}

int tree::sm_count() {
    static int count[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (!count[dev] && cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    return count[dev];
}

int tree::merge(const TreeParams& p, int hd, int rows, int tile, int grid, bool wide, int zero_tail, cudaStream_t st) {
    const long long n = (long long)p.N * p.H;
#define MERGE(HD_, W_)                                                                                                                  \
    return kb_launch_dep(tree_merge_kernel<HD_, W_>, dim3((unsigned)((n + 8 / W_ - 1) / (8 / W_))), dim3(256), 0, st, p, rows, tile, grid, zero_tail)
    if (hd == 128) {
        if (wide) MERGE(128, 8);
        MERGE(128, 1);
    }
    if (wide) MERGE(64, 8);
    MERGE(64, 1);
#undef MERGE
}

namespace {

struct Plan {
    int rows, tile, grid;
    bool wide;
};
// Which kernel, and how many CTAs: one per tile, at most what fits the GPU at once (one per SM for the 128-row kernel, two for the
// others).
Plan plan_for(int B, int N, int n_kv, int G, int max_q, int max_ctx, bool fp8) {
    Plan pl;
    const int most_rows = max_q * G;
    pl.rows = most_rows <= 16 ? 16 : most_rows <= 32 ? 32 : 128;
    pl.tile = pl.rows == 128 ? 128 : WARPS * (fp8 ? 32 : 16);
    const long long blocks = B + (long long)N * G / pl.rows;                            // units per KV head, at most
    const long long one = (most_rows + pl.rows - 1) / pl.rows;
    const long long units = n_kv * (blocks < B * one ? blocks : B * one), tiles = units * ((max_ctx + pl.tile - 1) / pl.tile);
    const long long most = (pl.rows == 128 ? 1ll : 2ll) * sm_count();
    pl.grid = (int)(tiles < most ? tiles : most);
    pl.wide = pl.grid > 8 * units;                     // parts per unit: one warp per row walks up to about eight of them
    return pl;
}

template <bool FP8, int HD, int MI>
int launch_tree(const CUtensorMap& tmK, const CUtensorMap& tmV, const TreeParams& p, const Plan& pl, cudaStream_t st) {
    static bool flags[64] = {};
    bool* set = kb_device_flag(flags);
    if (!set) return 7;
    if (!*set) {
        if (cudaFuncSetAttribute(tree_attn_kernel<FP8, HD, MI>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<FP8, HD, MI>::SMEM) != cudaSuccess) return 7;
        *set = true;
    }
    return kb_launch_dep(tree_attn_kernel<FP8, HD, MI>, dim3(pl.grid), dim3(THREADS), Cfg<FP8, HD, MI>::SMEM, st, tmK, tmV, p);
}

}  // namespace

// Floats of workspace that kb_tree_attn wants, 0 where the call is not one for it (the plain form takes it).
KB_API long long kb_tree_attn_floats(int N, int B, int H, int n_kv, int hd, int max_q, int max_ctx, int num_pages, int fp8) {
    if (N < 1 || B < 1 || B > MAX_B || n_kv < 1 || H < n_kv || H % n_kv || (hd != 64 && hd != 128) || max_q < 1 || max_q > 64 || max_ctx < 1 ||
        (long long)num_pages * n_kv * PAGE > 0x7fffffffll || (long long)N * H > 0x7fffffffll ||
        (long long)B * n_kv * ((max_q * (long long)(H / n_kv) + 15) / 16) * ((max_ctx + 63ll) / 64) > 0x7fffffffll / 1024)
        return 0;
    const Plan pl = plan_for(B, N, n_kv, H / n_kv, max_q, max_ctx, fp8 != 0);
    return 2ll * pl.grid * pl.rows * (hd + 2) + B + 4;
}

// As kb_tree_attn_plain for bf16 and heads of 64 and 128; query rows 16-byte, output rows 8-byte aligned; `work` has kb_tree_attn_floats
// floats (16-byte aligned).
KB_API int kb_tree_attn(const void* q, long long q_stride, const void* k, const void* ke, const void* v, const void* ve, const int* table, int max_pages,
                        int num_pages, const int* ctx_lens, const int* cu, int B, const long long* masks, void* out, long long out_stride, int N,
                        int H, int n_kv, int hd, int max_q, int max_ctx, float scale, int zero_tail, float* work, long long work_floats, int* status,
                        cudaStream_t st) {
    const bool fp8 = ke != nullptr;
    if ((ke == nullptr) != (ve == nullptr) || q_stride % 8 || out_stride % 4 || max_pages < 1 || num_pages < 1 || !status ||
        ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)ke | (uintptr_t)ve | (uintptr_t)work) % 16 || (uintptr_t)out % 8)
        return 5;
    const long long need = kb_tree_attn_floats(N, B, H, n_kv, hd, max_q, max_ctx, num_pages, fp8);
    if (need == 0 || work_floats < need) return 5;
    const Plan pl = plan_for(B, N, n_kv, H / n_kv, max_q, max_ctx, fp8);
    CUtensorMap tmK, tmV;
    const long long rows = (long long)num_pages * n_kv * PAGE;
    int r = page_map(&tmK, k, rows, hd, fp8, pl.rows == 128);
    if (!r) r = page_map(&tmV, v, rows, hd, fp8, pl.rows == 128);
    if (r) return r;
    TreeParams p;
    p.q = (const bf16*)q;
    p.q_stride = q_stride;
    p.ke = (const uint8_t*)ke;
    p.ve = (const uint8_t*)ve;
    p.table = table;
    p.ctx_lens = ctx_lens;
    p.cu = cu;
    p.masks = masks;
    p.out = (bf16*)out;
    p.out_stride = out_stride;
    p.part_o = work;
    p.part_ml = work + 2ll * pl.grid * pl.rows * hd;
    p.uoff = reinterpret_cast<int*>(p.part_ml + 2ll * pl.grid * pl.rows * 2);
    p.max_pages = max_pages;
    p.num_pages = num_pages;
    p.B = B;
    p.N = N;
    p.H = H;
    p.G = H / n_kv;
    p.n_kv = n_kv;
    p.max_q = max_q;
    p.max_ctx = max_ctx;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.status = status;
#define TREE(F, D) r = pl.rows == 16 ? launch_tree<F, D, 1>(tmK, tmV, p, pl, st) : launch_tree<F, D, 2>(tmK, tmV, p, pl, st)
    if (pl.rows == 128) r = launch_tile(tmK, tmV, p, hd, fp8, pl.grid, st);
    else if (fp8 && hd == 128) TREE(true, 128);
    else if (fp8) TREE(true, 64);
    else if (hd == 128) TREE(false, 128);
    else TREE(false, 64);
#undef TREE
    return r ? r : merge(p, hd, pl.rows, pl.tile, pl.grid, pl.wide, zero_tail, st);
}
