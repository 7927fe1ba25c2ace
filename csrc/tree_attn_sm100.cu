// Attention of drafted tokens over the paged cache for heads of 64 and 128 in bf16, pages in bf16 or 8 bits (cache_fp8.cu).  What a row
// sees is defined in tree_attn.cu.
//
// What bounds it.  A cached row is used by the (drafted token, query head) rows of its KV head only - 1 to a few hundred - so the
// cache's bytes bound the call, and above ~100 rows the tensor cores do.  Each (sequence, KV head) has its n * G query rows as the
// M side of `mma.sync.m16n8k16` tiles (16 of them per unit of work), cached tokens are the N side of the score product and the K side of
// the output product; probabilities go from accumulators to operands in registers.  Calls with more rows per KV head
// (`plan_for` below) take tree_attn_tile_sm100.cu.  Measured: 64 x 1 tokens over 2048, 8 bits, 24 query and 8 KV heads, 51 us, 4.0 TB/s, with the issue slots at
// 44 %, DRAM at 50 and the tensor cores at 27 %: 12 warps per SM, what 168 registers admit, do not cover a step's latencies.
//
// Work.  A unit is (sequence, KV head, block of rows); its tiles are TILE tokens of the context.  All units' tiles form one line
// that is cut into equal parts, one per worker, so that ragged contexts and one long context load the GPU alike.  Here a worker is a
// warp (in tree_attn_tile_sm100.cu a CTA): it copies its tiles into a ring of its own, 16 bytes per lane, and waits for no other warp.
// A unit that lies inside a part is finished there, the others leave partial results (unnormalised output, maximum, sum per row)
// that the merge kernel puts together.  A worker has at most two such partial units: the one it enters with (slot 0) and the one it
// leaves with (slot 1).  Short contexts are cut differently: a block of threads per unit, no merge (DIRECT below).
//
// 8-bit pages.  Codes become f16 (exact) on the way to the tensor cores.  Keys: the score's accumulator is scaled by the token's power of two.
// Values: the probability is scaled by the token's power of two relative to E, the largest seen so far by the warp, times 2^4, and
// rounded to f16; the output is kept in units of 2^(E - 4).  Maxima are renewed when a score exceeds them by 2^11, so f16's largest is
// 2^15; a scaled probability keeps eleven bits down to 2^-18 and is off by at most 2^-29 below.
// Values whose powers lie more than 2^SPREAD apart: added in fp32 like values that are not finite, so that a token that a row does not see or gives
// no weight takes nothing from it, however large it is.
// Queries become f16 with a power of two per row taken out, which brings the largest number to [1, 2): exact from 2^-17 on, off by at most 2^-25 below.
// bf16 pages: queries as they are, probabilities rounded to bf16, since both operands of a product have one type (16 x 16 tokens over 4000: off by 0.0023
// of the result in 64 bits, where rounding the result alone leaves 0.0017).  Scores, maxima, sums and outputs are fp32.
#include "tree_attn.cuh"

namespace {

using namespace tree;

constexpr int WARPS = 4, THREADS = WARPS * 32, CTAS = 3;     // CTAs per SM: what registers and shared memory admit

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
template <bool FP8, int HD>
struct Cfg {
    static constexpr int ROWS = 16;
    static constexpr int TILE = FP8 || HD == 64 ? 32 : 16;     // tokens of a step
    static constexpr int PAGES = TILE / PAGE;
    static constexpr int ROW_BYTES = FP8 ? HD : 2 * HD;
    static constexpr int PAGE_BYTES = PAGE * ROW_BYTES;
    static constexpr int STAGE = 2 * PAGES * PAGE_BYTES;               // keys, then values
    static constexpr int NST = FP8 && HD == 64 ? 4 : 2;
    // Where 16-byte piece `i` of a page's rows goes: rows of 64, 128 or 256 bytes (two halves of 128), each group of eight 16-byte places
    // of the banks permuted by the row, so that ldmatrix meets all banks.
    __device__ static __forceinline__ uint32_t place(int i) {
        if (ROW_BYTES == 64) return (i >> 2) * 64 + (((i & 3) ^ ((i >> 3) & 3)) << 4);
        if (ROW_BYTES == 128) return (i >> 3) * 128 + (((i & 7) ^ ((i >> 3) & 7)) << 4);
        return ((i >> 3) & 1) * 2048 + (i >> 4) * 128 + (((i & 7) ^ ((i >> 4) & 7)) << 4);
    }
    // place(32 i + lane) from place(lane)
    __device__ static __forceinline__ uint32_t place_next(uint32_t at, int i) {
        if (ROW_BYTES == 64) return at + i * 512;
        if (ROW_BYTES == 128) return (at ^ ((i & 1) << 6)) + i * 512;
        return (at ^ ((i & 3) << 5)) + i * 256;
    }
    static constexpr int RING = WARPS * NST * STAGE;
    static constexpr int EXPS = FP8 ? WARPS * NST * 2 * TILE : 0;      // exponents of a stage: keys, then values
    static constexpr int FACT = FP8 ? WARPS * 2 * TILE * 4 : 0;        // the step's factors as fp32
    static constexpr int SMEM = RING + EXPS + FACT;
};

// n rows of G heads from row c0 on, head h * G -> zero, by all threads of the block.
__device__ __forceinline__ void zero_rows(const TreeParams& p, int c0, int n, int head, int dims) {
    for (int row = 0; row < n; ++row) {
        bf16* dst = p.out + (long long)(c0 + row) * p.out_stride + (long long)head;
        for (int d = threadIdx.x * 4; d < dims; d += THREADS * 4) *reinterpret_cast<uint2*>(dst + d) = make_uint2(0u, 0u);
    }
}

// DIRECT: a block of threads per unit, whose tiles its warps share; nothing is left for a merge.  Else the line of tiles of all units.
template <bool FP8, int HD, bool DIRECT>
__global__ void __launch_bounds__(THREADS, CTAS)
tree_attn_kernel(const TreeParams p) {
    using C = Cfg<FP8, HD>;
    constexpr int TILE = C::TILE, NT = TILE / 8, KS = HD / 16;
    // log2 units: when a maximum is renewed; 8-bit pages: probabilities carry 2^UP, and f16 holds 2^(GROW + UP)
    constexpr int UP = 4;
    constexpr float GROW = FP8 ? 11.f : 20.f;
    extern __shared__ __align__(128) uint8_t ring_all[];
    uint8_t* exps_all = ring_all + C::RING;
    float* fact_all = reinterpret_cast<float*>(exps_all + C::EXPS);
    __shared__ int uoff[MAX_B + 1];
    __shared__ int wsum[WARPS];
    __shared__ uint32_t there[WARPS][C::NST];          // bit per page of a stage: loaded
    __shared__ float2 wml[WARPS][C::ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, qd = lane & 3;
    kb_dep_wait();
    kb_dep_trigger();
    const int worker = blockIdx.x * WARPS + warp;
    Segment whole_unit = {};                           // (DIRECT)
    if constexpr (DIRECT) {
        const int bh = blockIdx.x / p.row_blocks, b = bh / p.n_kv, end = p.cu ? p.cu[p.B] : p.B;
        whole_unit.b = b;
        whole_unit.h = bh % p.n_kv;
        whole_unit.rb = blockIdx.x % p.row_blocks;
        if (p.zero_tail) {                             // rows behind the last sequence, and in front of the first
            for (int n = max(end, 0) + blockIdx.x; n < p.N; n += gridDim.x) zero_rows(p, n, 1, 0, p.H * HD);
            for (int n = blockIdx.x; p.cu && n < min(p.cu[0], p.N); n += gridDim.x) zero_rows(p, n, 1, 0, p.H * HD);
        }
        const bool first = whole_unit.rb == 0;
        const int2 sp = span_of(p, b, first && whole_unit.h == 0 && threadIdx.x == 0);
        if (sp.x == 0) {
            const int c0 = max(p.cu ? p.cu[b] : b, 0), c1 = min(p.cu ? p.cu[b + 1] : b + 1, p.N);
            if (first) zero_rows(p, c0, c1 - c0, whole_unit.h * p.G * HD, p.G * HD);
            return;
        }
        if (whole_unit.rb * C::ROWS >= sp.x * p.G) return;
        whole_unit.n = sp.x;
        whole_unit.ctx = sp.y;
        whole_unit.T = (sp.y + TILE - 1) / TILE;
    } else {
        count_tiles<C::ROWS, TILE, THREADS>(p, uoff, wsum);
        if (uoff[p.B] == 0) return;
    }
    const int2 part = DIRECT ? make_int2(whole_unit.T * warp / WARPS, whole_unit.T * (warp + 1) / WARPS) : part_of_line(uoff[p.B], worker, gridDim.x * WARPS);
    const int lo = part.x, hi = part.y;
    auto segment = [&](int x) {
        if constexpr (!DIRECT) return segment_at<C::ROWS, TILE>(p, uoff, x, hi);
        Segment s = whole_unit;
        s.t0 = x;
        s.t1 = hi;
        return s;
    };

    // ---- this warp's ring: item k is tile lo + k
    uint8_t* ring = ring_all + (size_t)warp * C::NST * C::STAGE;
    uint8_t* exps = exps_all + warp * C::NST * 2 * TILE;
    const Segment unit = segment(DIRECT ? lo : min(lo, uoff[p.B] - 1));        // the first unit of the part
    Segment ps = unit;
    // Whether the block's four parts lie in one unit: their results then meet in shared memory, and the merge has a quarter of the parts.
    const int2 cta_first = DIRECT ? make_int2(0, 0) : part_of_line(uoff[p.B], blockIdx.x * WARPS, gridDim.x * WARPS);
    const int2 cta_last = DIRECT ? make_int2(0, unit.T) : part_of_line(uoff[p.B], blockIdx.x * WARPS + WARPS - 1, gridDim.x * WARPS);
    const bool together = DIRECT || cta_last.y > 0 && cta_first.x >= lo - unit.t0 && cta_last.y <= lo - unit.t0 + unit.T;
    int px = lo, pfirst = lo;                          // next tile to issue; tile at which ps begins
    int next_page = -1;                                // lane l < PAGES: page number of the next item (fetched one item ahead)
    auto fetch_page = [&]() {
        if (px >= hi) return;
        if (px - pfirst >= ps.t1 - ps.t0) {
            ps = segment(px);
            pfirst = px;
        }
        const int tok = (ps.t0 + px - pfirst) * TILE + lane * PAGE;
        next_page = -2;                                // nothing to load
        if (lane < C::PAGES && tok < ps.ctx) next_page = p.table[(long long)ps.b * p.max_pages + tok / PAGE];
    };
    fetch_page();
    const uint32_t my_place = C::place(lane);
    auto copy_page = [&](uint32_t dst, int st, int pg) {
        const uint32_t cell = (uint32_t)__shfl_sync(0xffffffffu, next_page, pg) * (uint32_t)p.n_kv + (uint32_t)ps.h;
        const uint8_t *k = p.k + (unsigned long long)cell * C::PAGE_BYTES + lane * 16, *v = p.v + (unsigned long long)cell * C::PAGE_BYTES + lane * 16;
#pragma unroll
        for (int i = 0; i < C::PAGE_BYTES / 512; ++i) {
            const uint32_t at = dst + pg * C::PAGE_BYTES + C::place_next(my_place, i);
            copy16(at, k + i * 512);
            copy16(at + C::PAGES * C::PAGE_BYTES, v + i * 512);
        }
        if (FP8 && lane < 2) copy16(smem_u32(exps + st * 2 * TILE + lane * TILE + pg * PAGE), (lane ? p.ve : p.ke) + (unsigned long long)cell * PAGE);
    };
    auto issue = [&]() {                               // loads item px, then looks up the page numbers of the one after it
        if (px < hi) {
            const int st = (px - lo) % C::NST;
            const bool good = (uint32_t)next_page < (uint32_t)p.num_pages;
            const uint32_t have = __ballot_sync(0xffffffffu, lane < C::PAGES && good);
            if (lane == 0) there[warp][st] = have;
            const uint32_t dst = smem_u32(ring + st * C::STAGE);
            if (have == (1u << C::PAGES) - 1u) {
#pragma unroll
                for (int pg = 0; pg < C::PAGES; ++pg) copy_page(dst, st, pg);
            } else {
                if (lane < C::PAGES && next_page != -2 && !good && p.status) atomicMax(p.status, (int)KB_BAD_INDEX);
#pragma unroll 1
                for (int pg = 0; pg < C::PAGES; ++pg)
                    if (have >> pg & 1u) copy_page(dst, st, pg);
            }
            ++px;
            fetch_page();
        }
        copy_commit();                                 // (an empty group behind the last item: the count of groups goes on)
    };
    for (int i = 0; i < C::NST; ++i) issue();

    for (int x = lo; x < hi;) {
        const Segment sg = segment(x);
        const int row0 = sg.rb * C::ROWS, M = sg.n * p.G, prefix = sg.ctx - sg.n;
        const int c0 = p.cu ? p.cu[sg.b] : sg.b;
        // ---- the unit's queries as A fragments
        uint32_t qa[KS][4];
        float rs[2];                                   // 8-bit pages: the power of two taken out of rows r, r + 8
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int R = row0 + hf * 8 + r;
            const bf16* src = p.q + (long long)(c0 + R / p.G) * p.q_stride + (long long)(sg.h * p.G + R % p.G) * HD;
            uint2 raw[KS];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                raw[ks] = make_uint2(0u, 0u);
                if (R < M) {
                    if constexpr (FP8) raw[ks] = *reinterpret_cast<const uint2*>(src + ks * 16 + 4 * qd);
                    else raw[ks] = make_uint2(*reinterpret_cast<const uint32_t*>(src + ks * 16 + 2 * qd), *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8 + 2 * qd));
                }
            }
            rs[hf] = 1.f;
            if constexpr (FP8) {                       // take a power of two out of the row, then f16
                uint32_t big = 0;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) big = max(big, max(max(raw[ks].x & 0x7fffu, (raw[ks].x >> 16) & 0x7fffu), max(raw[ks].y & 0x7fffu, (raw[ks].y >> 16) & 0x7fffu)));
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                const int e = min(max((int)(big >> 7), Q_LEAST), 253);     // biased exponent of the largest number
                const float inv = pow2_biased(254 - e);
                rs[hf] = pow2_biased(e);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    raw[ks] = make_uint2(pack_f16(__uint_as_float(raw[ks].x << 16) * inv, __uint_as_float(raw[ks].x & 0xffff0000u) * inv),
                                         pack_f16(__uint_as_float(raw[ks].y << 16) * inv, __uint_as_float(raw[ks].y & 0xffff0000u) * inv));
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                qa[ks][hf] = raw[ks].x;
                qa[ks][2 + hf] = raw[ks].y;
            }
        }
        float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        int E = 0, low = 255;                          // biased exponent of the output's unit; the smallest of the values so far
        constexpr int APART = -1;                      // for E: the output is in units of one, values are added in fp32
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        for (int t = sg.t0; t < sg.t1; ++t, ++x) {
            const int st = (x - lo) % C::NST;
            copy_wait<C::NST - 1>();
            __syncwarp();
            const int base = t * TILE;
            const uint32_t have = there[warp][st];
            if (have) {
                const uint32_t kb = smem_u32(ring + (size_t)st * C::STAGE), vb = kb + C::PAGES * C::PAGE_BYTES;
                uint32_t valid = 0;                    // tokens of the step that exist
#pragma unroll
                for (int i = 0; i < C::PAGES; ++i) valid |= (have >> i & 1u) * (0xffffu << (16 * i));
                if (base + TILE > sg.ctx) valid &= 0xffffffffu >> (32 - (sg.ctx - base));
                const bool whole = valid == (TILE == 32 ? 0xffffffffu : 0xffffu), drafts = base + TILE > prefix;
                float* fk = fact_all + warp * 2 * TILE;
                float grow = 1.f;                      // factor of the output's change of unit
                if constexpr (FP8) {
                    const uint8_t* e = exps + st * 2 * TILE;
                    const int ek = e[lane], ev = e[TILE + lane];
                    const bool counts = (valid >> lane & 1u) && ev != 255;
                    const int top = (int)__reduce_max_sync(0xffffffffu, counts ? (unsigned)ev : 0u);
                    low = min(low, (int)__reduce_min_sync(0xffffffffu, counts ? (unsigned)ev : 255u));
                    if (E != APART && max(top, E) - low > SPREAD) {
                        grow = exp2f((float)(E - 127 - UP));               // (zero ahead of the first token: so is the output)
                        E = APART;
                    }
                    if (E != APART && top > E) {
                        grow = exp2f((float)(E - top));
                        E = top;
                    }
                    fk[lane] = pow2_biased(ek) * p.scale_log2;
                    fk[TILE + lane] = counts && E != APART ? __uint_as_float((uint32_t)(ev - E + UP + 127) << 23) : 1.f;
                    __syncwarp();
                }
                // ---- scores
                float s[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
                if constexpr (FP8) {
                    const uint32_t row = kb + lane * HD;                   // ldmatrix: matrix i holds the tokens of n tile i
                    const int sw = HD == 128 ? lane & 7 : (lane >> 1) & 3;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        uint32_t c[4];
                        ldsm_x4(row + ((ks ^ sw) << 4), c);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t b0, b1;
                            codes_to_f16(c[j], b0, b1);
                            mma<true>(s[j], qa[ks], b0, b1);
                        }
                    }
                } else {
                    const int tok = (lane & 7) + (lane >> 4) * 8, sub = (lane >> 3) & 1;
#pragma unroll
                    for (int pg = 0; pg < C::PAGES; ++pg)
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) {
                            const int ch = ks * 2 + sub;
                            uint32_t b[4];
                            ldsm_x4(kb + pg * C::PAGE_BYTES + (ch >> 3) * 2048 + tok * 128 + (((ch & 7) ^ (tok & 7)) << 4), b);
                            mma<false>(s[2 * pg], qa[ks], b[0], b[1]);
                            mma<false>(s[2 * pg + 1], qa[ks], b[2], b[3]);
                        }
                }
                // In log2 units (8-bit pages: but for the row's power of two, which rounds nothing) before anything is hidden or subtracted: a scale
                // that vanishes would make NaN of a hidden score, one inside the subtraction would leave its product's rounding, which for
                // scores from 2^32 on is more than an exponential holds
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float2 f = make_float2(p.scale_log2, p.scale_log2);
                    if constexpr (FP8) f = *reinterpret_cast<const float2*>(fk + 8 * j + 2 * qd);
                    s[j][0] *= f.x;
                    s[j][1] *= f.y;
                    s[j][2] *= f.x;
                    s[j][3] *= f.y;
                }
                // ---- what is not seen: places that hold no token, and drafted tokens the row's mask does not name
                uint32_t odd = FP8 && E == APART ? valid : 0u;             // tokens kept out of the product: drafted ones whose values are not finite, or all
                uint32_t seen[2] = {~0u, ~0u};         // bit t: the row sees token t of the step
                if (!whole || drafts) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const int i = min((row0 + hf * 8 + r) / p.G, sg.n - 1);
                        seen[hf] = (uint32_t)sees(p, c0, i, base - prefix) & valid;
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            const uint32_t two = seen[hf] >> (8 * j + 2 * qd);
                            if (!(two & 1u)) s[j][2 * hf] = -INFINITY;
                            if (!(two & 2u)) s[j][2 * hf + 1] = -INFINITY;
                        }
                    }
                    if (drafts) {
                        bool bad = false;
                        if (lane < TILE && (valid >> lane & 1u) && base + lane >= prefix) {
                            const uint8_t* page = ring + (size_t)st * C::STAGE + (C::PAGES + lane / PAGE) * C::PAGE_BYTES;
#pragma unroll 1
                            for (int c = 0; c < C::ROW_BYTES / 16; ++c) {
                                const uint4 v = *reinterpret_cast<const uint4*>(page + C::place((lane % PAGE) * (C::ROW_BYTES / 16) + c));
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int q = 0; q < 4; ++q)
                                    bad |= FP8 ? __vcmpeq4(w[q] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0u : __vcmpeq2(w[q] & 0x7f807f80u, 0x7f807f80u) != 0u;
                            }
                        }
                        odd |= __ballot_sync(0xffffffffu, bad);
                    }
                }
                // ---- softmax against a maximum that is renewed only when a score exceeds it by more than GROW
                float mx[2];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    mx[hf] = fmaxf(s[0][2 * hf], s[0][2 * hf + 1]);
#pragma unroll
                    for (int j = 1; j < NT; ++j) mx[hf] = fmaxf(mx[hf], fmaxf(s[j][2 * hf], s[j][2 * hf + 1]));
                    if constexpr (FP8) mx[hf] *= rs[hf];
                }
                if (__any_sync(0xffffffffu, mx[0] > m[0] + GROW || mx[1] > m[1] + GROW || (FP8 && grow != 1.f))) {
                    float f[2];
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 1));
                        mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 2));
                        const float mn = fmaxf(m[hf], mx[hf]);
                        f[hf] = mn == -INFINITY ? 1.f : exp2f(m[hf] - mn);
                        m[hf] = mn;
                        l[hf] *= f[hf];
                        f[hf] *= grow;
                    }
#pragma unroll
                    for (int j = 0; j < HD / 8; ++j) {
                        o[j][0] *= f[0];
                        o[j][1] *= f[0];
                        o[j][2] *= f[1];
                        o[j][3] *= f[1];
                    }
                }
                uint32_t pa[TILE / 16][4];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const float at = m[hf] == -INFINITY ? 0.f : m[hf];
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float a = exp2f(FP8 ? fmaf(s[j][2 * hf], rs[hf], -at) : s[j][2 * hf] - at);
                        float z = exp2f(FP8 ? fmaf(s[j][2 * hf + 1], rs[hf], -at) : s[j][2 * hf + 1] - at);
                        l[hf] += a + z;
                        if constexpr (FP8) {
                            const float2 w = *reinterpret_cast<const float2*>(fk + TILE + 8 * j + 2 * qd);
                            a *= w.x;
                            z *= w.y;
                        }
                        s[j][2 * hf] = a;
                        s[j][2 * hf + 1] = z;
                        pa[j >> 1][(j & 1) * 2 + hf] = FP8 ? pack_f16(a, z) : pack_bf16(a, z);
                    }
                }
                if (!whole || odd) {
                    // Values that must not enter the product: what the cache holds in places without a token, and the odd tokens, which are
                    // added row by row (never in normal use)
                    uint8_t* pages = ring + (size_t)st * C::STAGE + C::PAGES * C::PAGE_BYTES;
                    volatile float kept[NT][4];        // (indexed by the token: in local memory, here only)
                    if (odd)
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) kept[j][e] = s[j][e];
#pragma unroll 1
                    for (uint32_t left = odd; left; left &= left - 1u) {
                        const int tk = __ffs(left) - 1, src = (lane & ~3) | ((tk & 7) >> 1), tr = tk % PAGE;
                        const uint8_t* page = pages + (tk / PAGE) * C::PAGE_BYTES;
                        const float unit = FP8 && E == APART ? pow2_biased(exps[st * 2 * TILE + TILE + tk]) : 1.f;
                        float pv[2];
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) pv[hf] = __shfl_sync(0xffffffffu, kept[tk >> 3][2 * hf + (tk & 1)], src);
#pragma unroll
                        for (int j = 0; j < HD / 8; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int d = FP8 ? (j >> 1) * 16 + 4 * qd + 2 * e + (j & 1) : 8 * j + 2 * qd + e, byte = FP8 ? d : 2 * d;
                                const uint8_t* at = page + C::place(tr * (C::ROW_BYTES / 16) + byte / 16) + byte % 16;
                                const float v = FP8 ? __half2float(__half(__nv_cvt_fp8_to_halfraw(*at, __NV_E4M3))) * unit : __bfloat162float(*reinterpret_cast<const bf16*>(at));
                                if (seen[0] >> tk & 1u) o[j][e] += pv[0] * v;
                                if (seen[1] >> tk & 1u) o[j][2 + e] += pv[1] * v;
                            }
                    }
                    __syncwarp();
                    if (lane < TILE && !(valid >> lane & ~(odd >> lane) & 1u))
#pragma unroll 1
                        for (int c = 0; c < C::ROW_BYTES / 16; ++c)
                            *reinterpret_cast<uint4*>(pages + (lane / PAGE) * C::PAGE_BYTES + C::place((lane % PAGE) * (C::ROW_BYTES / 16) + c)) = make_uint4(0u, 0u, 0u, 0u);
                    __syncwarp();
                }
                // ---- output
                const int vtok = (lane & 7) + ((lane >> 3) & 1) * 8, vsub = lane >> 4;
#pragma unroll
                for (int kk = 0; kk < TILE / 16; ++kk) {
                    const uint32_t page = vb + kk * C::PAGE_BYTES;
                    if constexpr (FP8) {
                        const uint32_t row = page + vtok * HD;
                        const int sw = HD == 128 ? vtok & 7 : (vtok >> 1) & 3;
#pragma unroll
                        for (int c = 0; c < HD / 16; c += 2) {
                            uint32_t v[4];
                            ldsm_x4_t(row + (((c + vsub) ^ sw) << 4), v);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                uint32_t e0, o0, e1, o1;                   // even and odd head dimensions of the chunk
                                codes_to_f16(__byte_perm(v[2 * i], 0, 0x3120), e0, o0);
                                codes_to_f16(__byte_perm(v[2 * i + 1], 0, 0x3120), e1, o1);
                                mma<true>(o[2 * (c + i)], pa[kk], e0, e1);
                                mma<true>(o[2 * (c + i) + 1], pa[kk], o0, o1);
                            }
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < HD / 16; ++j) {
                            const int ch = j * 2 + vsub;
                            uint32_t v[4];
                            ldsm_x4_t(page + (ch >> 3) * 2048 + vtok * 128 + (((ch & 7) ^ (vtok & 7)) << 4), v);
                            mma<false>(o[2 * j], pa[kk], v[0], v[1]);
                            mma<false>(o[2 * j + 1], pa[kk], v[2], v[3]);
                        }
                    }
                }
            }
            __syncwarp();                              // every lane has read the stage
            issue();
        }
        // ---- the unit's rows, as far as this warp has them
        const bool done = !together && sg.t0 == 0 && sg.t1 == sg.T;
        const long long slot = 2ll * worker + (sg.t0 == 0);
        float* part_o = p.part_o + slot * C::ROWS * HD;
        if (together) {                                // the ring is idle now: [16][HD] floats at its start
            copy_wait<0>();
            __syncwarp();
            part_o = reinterpret_cast<float*>(ring);
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
            const int row = hf * 8 + r, R = row0 + row;
            if (R >= M) continue;
            float g = FP8 && E != APART ? pow2_biased(E) * (1.f / (1 << UP)) : 1.f;    // 2^(E - 127 - UP)
            if (done) g *= l[hf] == 0.f ? 0.f : 1.f / l[hf];
            bf16* dst = p.out + (long long)(c0 + R / p.G) * p.out_stride + (long long)(sg.h * p.G + R % p.G) * HD;
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) {
                if constexpr (FP8) {                   // dimensions 4 qd .. 4 qd + 3 of a chunk of 16: evens in one tile, odds in the other
                    if (j & 1) continue;
                    const int d = j * 8 + 4 * qd;
                    const float a = o[j][2 * hf] * g, b = o[j + 1][2 * hf] * g, c = o[j][2 * hf + 1] * g, e = o[j + 1][2 * hf + 1] * g;
                    if (done) *reinterpret_cast<uint2*>(dst + d) = make_uint2(pack_bf16(a, b), pack_bf16(c, e));
                    else *reinterpret_cast<float4*>(part_o + row * HD + d) = make_float4(a, b, c, e);
                } else {
                    const int d = j * 8 + 2 * qd;
                    const float a = o[j][2 * hf] * g, b = o[j][2 * hf + 1] * g;
                    if (done) *reinterpret_cast<uint32_t*>(dst + d) = pack_bf16(a, b);
                    else *reinterpret_cast<float2*>(part_o + row * HD + d) = make_float2(a, b);
                }
            }
            if (!done && qd == 0) {
                if (together) wml[warp][row] = make_float2(m[hf], l[hf]);
                else *reinterpret_cast<float2*>(p.part_ml + (slot * C::ROWS + row) * 2) = make_float2(m[hf], l[hf]);
            }
        }
    }
    copy_wait<0>();
    if (!together) return;
    __syncthreads();
    const int x0 = DIRECT ? 0 : cta_first.x - (lo - unit.t0), x1 = DIRECT ? unit.T : cta_last.y - (lo - unit.t0);      // the block's tiles of the unit
    auto idle = [&](int w) { return DIRECT && unit.T * w / WARPS == unit.T * (w + 1) / WARPS; };       // a warp without a tile has left nothing
    const bool done = x0 == 0 && x1 == unit.T;
    const long long slot = 2ll * blockIdx.x * WARPS + (x0 == 0);
    const int M = unit.n * p.G - unit.rb * C::ROWS, c0 = p.cu ? p.cu[unit.b] : unit.b;
    for (int i = threadIdx.x; i < min(M, C::ROWS) * (HD / 4); i += THREADS) {
        const int row = i / (HD / 4), d = i % (HD / 4) * 4;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
            if (!idle(w)) top = fmaxf(top, wml[w][row].x);
        const float at = top == -INFINITY ? 0.f : top;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (idle(w)) continue;
            const float2 ml = wml[w][row];
            const float g = exp2f(ml.x - at);
            sum += ml.x == -INFINITY ? ml.y : ml.y * g;                    // a sum without a maximum is zero, or NaN and has to get through
            const float4 u = *reinterpret_cast<const float4*>(ring_all + (size_t)w * C::NST * C::STAGE + (row * HD + d) * 4);
            v.x += u.x * g;
            v.y += u.y * g;
            v.z += u.z * g;
            v.w += u.w * g;
        }
        if (done) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int R = unit.rb * C::ROWS + row;
            bf16* dst = p.out + (long long)(c0 + R / p.G) * p.out_stride + (long long)(unit.h * p.G + R % p.G) * HD + d;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
        } else {
            *reinterpret_cast<float4*>(p.part_o + (slot * C::ROWS + row) * HD + d) = v;
            if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * C::ROWS + row) * 2) = make_float2(top, sum);
        }
    }
}

// Puts the parts of a unit together; WPR warps share a row.  `per`: workers of a block; where all of a block's parts lie in the unit the
// block has left one part for them.  Rows of sequences without rows or tokens, and (zero_tail) rows behind the last sequence, become zero.
// ROW_MAJOR: parts are [rows][HD], else [HD / 4][rows][4].
template <int HD, int WPR, bool ROW_MAJOR>
__global__ void __launch_bounds__(WPR == 1 ? 256 : WPR * 32)
tree_merge_kernel(const TreeParams p, int ROWS, int TILE, int workers, int per, int zero_tail) {
    constexpr int RPB = WPR == 1 ? 8 : 1, EPL = HD / 32;       // rows per block; dimensions per lane
    __shared__ float so[WPR > 1 ? WPR : 1][HD], sml[WPR][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR;
    const long long row = (long long)blockIdx.x * RPB + warp / WPR;
    if (row >= (long long)p.N * p.H) {                 // (with several warps per row the whole block)
        kb_dep_wait();
        return;
    }
    // What the sequences are was known before the kernel ahead began (it lets this one start after its own wait)
    const int n = (int)(row / p.H), head = (int)(row % p.H), h = head / p.G;
    int b = n;
    if (p.cu) {                                        // sequences that end at or before row n
        b = 0;
        for (int i = lane; i < p.B; i += 32) b += p.cu[i + 1] <= n;
        b = __reduce_add_sync(0xffffffffu, b);
    }
    const int c0 = b < p.B ? (p.cu ? p.cu[b] : b) : 0, c1 = b < p.B ? (p.cu ? p.cu[b + 1] : b + 1) : 0;
    const bool inside = b < p.B && n >= c0 && n < c1;
    bf16* dst = p.out + (long long)n * p.out_stride + (long long)head * HD + lane * EPL;
    const int2 sp = inside ? span_of(p, b, false) : make_int2(0, 0);
    kb_dep_wait();
    kb_dep_trigger();
    if (sp.x == 0) {
        if ((inside || zero_tail) && sub == 0)
#pragma unroll
            for (int e = 0; e < EPL; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = 0u;
        return;
    }
    const int Rl = (n - c0) * p.G + head % p.G, rbs = (sp.x * p.G + ROWS - 1) / ROWS, T = (sp.y + TILE - 1) / TILE;
    const long long total = p.uoff[p.B], s0 = p.uoff[b] + (long long)(h * rbs + Rl / ROWS) * T;
    const long long parts = min((long long)workers, total);
    const int first = (int)(((s0 + 1) * parts - 1) / total), last = (int)(((s0 + T) * parts - 1) / total);
    // blocks of the first and last part, and whether a block has left one part
    const int cA = first / per, cB = last / per;
    auto whole = [&](int c) {
        return (long long)(c + 1) * per <= parts && total * c * per / parts >= s0 && total * (c + 1) * per / parts <= s0 + T;
    };
    const bool wA = whole(cA), wB = whole(cB);
    if (wA && cA == cB && s0 == total * cA * per / parts && s0 + T == total * (cA + 1) * per / parts) return;      // finished by its block
    if (first == last && !wA) return;                  // finished by its worker
    const int head_n = wA ? 1 : min(last, cA * per + per - 1) - first + 1, mid_n = cB > cA ? cB - cA - 1 : 0;
    const int all = head_n + mid_n + (cB > cA ? (wB ? 1 : last - cB * per + 1) : 0);
    const int r = Rl % ROWS;
    float M = -INFINITY, L = 0.f, acc[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
    constexpr int U = 4;                               // parts in flight
    for (int k0 = sub; k0 < all; k0 += WPR * U) {
        float2 ml[U];
        float v[U][EPL];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * WPR;
            ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int e = 0; e < EPL; ++e) v[u][e] = 0.f;
            if (k < all) {
                const int j = k < head_n ? first + k : k < head_n + mid_n ? (cA + 1 + k - head_n) * per : cB * per + k - head_n - mid_n;
                const long long slot = 2ll * j + (j == first);
                ml[u] = *reinterpret_cast<const float2*>(p.part_ml + (slot * ROWS + r) * 2);
#pragma unroll
                for (int e = 0; e < EPL; e += 2) {
                    const int d = lane * EPL + e;
                    const float* src = p.part_o + (ROW_MAJOR ? (slot * ROWS + r) * HD + d : ((slot * (HD / 4) + d / 4) * ROWS + r) * 4 + d % 4);
                    *reinterpret_cast<float2*>(&v[u][e]) = *reinterpret_cast<const float2*>(src);
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
#pragma unroll 8
        for (int w = 1; w < WPR; ++w) top = fmaxf(top, sml[w][0]);
        const float at = top == -INFINITY ? 0.f : top;
        L = 0.f;
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
#pragma unroll 4
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

}  // namespace

int tree::sm_count() {
    static int count[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (!count[dev] && cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    return count[dev];
}

namespace {

struct Plan {
    int rows, tile, grid, workers, per_cta, merge_warps, row_blocks;       // row_blocks: > 0 where a block of threads takes a unit
};
// Which kernel, and how many CTAs: as many as there are tiles for, at most what fits the GPU at once.  The 128-row kernel pays for 128 rows
// whatever there are, this one for units of 16 rows, of which each reads the keys and values again.  Measured (us, this kernel / the 128-row one), 64
// sequences over 2048 tokens, four query heads per KV head, rows per KV head 16 / 32 / 48 / 64: 8-bit pages 64 / 158, 98 / 165, 141 / 172, 178 / 179;
// bf16 pages 89 / 114, 139 / 120, -, 237 / 136.  So: up to 48 rows on 8-bit pages, up to 16 on bf16 pages.
// The merge walks a unit's parts with one warp per row where there are about eight of them, else with 8 or 32: (us, 1 / 8 / 32 warps) one token of 64
// sequences over 2048 tokens 52 / 59 / 98, one of one sequence over 4000 tokens 20 / 13 / 14, of four over 8000 35 / 30 / 30.
// Short contexts: a block of threads per unit where the units run at once, which needs no count of tiles, no partial results and no merge.  (us, so / the line
// of tiles) one token, 24 query and 8 KV heads: 1 sequence over 250 tokens 8.2 / 11.1 (bf16), 500 10.5 / 11.7, 1000 15.3 / 12.8, 2000 24.9 / 11.8; 16 over 500
// 11.1 / 15.4, bf16 (32 tiles) 11.5 / 17.4; 50 over 1000 25.6 / 33.5, over 2000 40.6 / 45.7.  Up to 16 tiles, or 32 where there are at least 64 units; more would
// lose twice what it gains when one sequence is long and the others short.  That holds for many rows as well (us, so / the 128-row kernel): 8 sequences of 8
// drafted tokens, 24 rows, bf16, over 500 tokens 14.7 / 23.3; 4 of 64, 192 rows, 17.3 / 33.3 (8 bits), 22.8 / 29.6 (bf16).
Plan plan_for(int B, int N, int n_kv, int G, int hd, int max_q, int max_ctx, bool fp8) {
    Plan pl;
    const int most_rows = max_q * G, tile16 = fp8 || hd == 64 ? 32 : 16;
    const long long direct = (long long)B * n_kv * ((most_rows + 15) / 16);            // blocks of threads, one per unit of 16 rows
    const bool take = direct <= (long long)CTAS * sm_count() && max_ctx <= (direct >= 64 ? 32 : 16) * tile16;
    pl.rows = take || most_rows <= (fp8 ? 48 : 16) ? 16 : 128;
    pl.tile = pl.rows == 128 ? 128 : tile16;
    const long long blocks = B + (long long)N * G / pl.rows;                            // units per KV head, at most
    const long long one = (most_rows + pl.rows - 1) / pl.rows;
    const long long units = n_kv * (blocks < B * one ? blocks : B * one), tiles = units * ((max_ctx + pl.tile - 1) / pl.tile);
    pl.per_cta = pl.rows == 128 ? 1 : WARPS;
    const long long want = (tiles + pl.per_cta - 1) / pl.per_cta, most = (long long)(pl.rows == 128 ? 1 : CTAS) * sm_count();
    pl.grid = (int)(take ? direct : want < most ? want : most);
    pl.workers = take ? 0 : pl.grid * pl.per_cta;
    pl.row_blocks = take ? (int)one : 0;
    pl.merge_warps = pl.grid <= 8 * units ? 1 : pl.grid <= 64 * units ? 8 : 32;
    return pl;
}

// The merge always starts while the kernel ahead of it runs: it waits for it on the device.
template <int HD, int W, bool ROW_MAJOR>
int launch_merge(const TreeParams& p, const Plan& pl, int zero_tail, cudaStream_t st) {
    const long long n = (long long)p.N * p.H;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)(W == 1 ? (n + 7) / 8 : n));
    cfg.blockDim = dim3(W == 1 ? 256 : W * 32);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, tree_merge_kernel<HD, W, ROW_MAJOR>, p, pl.rows, pl.tile, pl.workers, pl.per_cta, zero_tail) == cudaSuccess) return 0;
    cudaGetLastError();
    return KB_LAUNCH_FAILED;
}
template <int HD, bool ROW_MAJOR>
int merge(const TreeParams& p, const Plan& pl, int zero_tail, cudaStream_t st) {
    return pl.merge_warps == 1   ? launch_merge<HD, 1, ROW_MAJOR>(p, pl, zero_tail, st)
           : pl.merge_warps == 8 ? launch_merge<HD, 8, ROW_MAJOR>(p, pl, zero_tail, st)
                                 : launch_merge<HD, 32, ROW_MAJOR>(p, pl, zero_tail, st);
}

template <bool FP8, int HD, bool DIRECT>
int launch_form(const TreeParams& p, const Plan& pl, cudaStream_t st) {
    static bool flags[64] = {};
    bool* set = kb_device_flag(flags);
    if (!set) return 7;
    if (!*set) {
        if (cudaFuncSetAttribute(tree_attn_kernel<FP8, HD, DIRECT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<FP8, HD>::SMEM) != cudaSuccess) return 7;
        *set = true;
    }
    return kb_launch_dep(tree_attn_kernel<FP8, HD, DIRECT>, dim3(pl.grid), dim3(THREADS), Cfg<FP8, HD>::SMEM, st, p);
}
template <bool FP8, int HD>
int launch_tree(const TreeParams& p, const Plan& pl, cudaStream_t st) {
    return pl.row_blocks ? launch_form<FP8, HD, true>(p, pl, st) : launch_form<FP8, HD, false>(p, pl, st);
}

}  // namespace

// Floats of workspace that kb_tree_attn wants (-1: none), 0 where the call is not one for it (the plain form takes it).
KB_API long long kb_tree_attn_floats(int N, int B, int H, int n_kv, int hd, int max_q, int max_ctx, int fp8) {
    if (N < 1 || B < 1 || B > MAX_B || n_kv < 1 || H < n_kv || H % n_kv || (hd != 64 && hd != 128) || max_q < 1 || max_q > 64 || max_ctx < 1 ||
        (long long)N * H > 0x7fffffffll ||
        (long long)B * n_kv * ((max_q * (long long)(H / n_kv) + 15) / 16) * ((max_ctx + 15ll) / 16) > 0x7fffffffll / 64)
        return 0;
    const Plan pl = plan_for(B, N, n_kv, H / n_kv, hd, max_q, max_ctx, fp8 != 0);
    return pl.row_blocks ? -1 : 2ll * pl.workers * pl.rows * (hd + 2) + B + 4;
}

// As kb_tree_attn_plain for bf16 and heads of 64 and 128; query rows 16-byte, output rows 8-byte aligned; `work` has kb_tree_attn_floats
// floats (16-byte aligned).
KB_API int kb_tree_attn(const void* q, long long q_stride, const void* k, const void* ke, const void* v, const void* ve, const int* table, int max_pages,
                        int num_pages, const int* ctx_lens, const int* cu, int B, const long long* masks, void* out, long long out_stride, int N,
                        int H, int n_kv, int hd, int max_q, int max_ctx, float scale, int zero_tail, float* work, long long work_floats, int* status,
                        cudaStream_t st) {
    const bool fp8 = ke != nullptr;
    if ((ke == nullptr) != (ve == nullptr) || !(scale > 0.f) || (long long)num_pages * n_kv > 0x7fffffffll || q_stride % 8 || out_stride % 4 || max_pages < 1 || num_pages < 1 || !status ||
        ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)ke | (uintptr_t)ve | (uintptr_t)work) % 16 || (uintptr_t)out % 8)
        return 5;
    const long long need = kb_tree_attn_floats(N, B, H, n_kv, hd, max_q, max_ctx, fp8);
    if (need == 0 || (need > 0 && (work_floats < need || !work))) return 5;
    const Plan pl = plan_for(B, N, n_kv, H / n_kv, hd, max_q, max_ctx, fp8);
    TreeParams p;
    p.q = (const bf16*)q;
    p.q_stride = q_stride;
    p.k = (const uint8_t*)k;
    p.v = (const uint8_t*)v;
    p.ke = (const uint8_t*)ke;
    p.ve = (const uint8_t*)ve;
    p.table = table;
    p.ctx_lens = ctx_lens;
    p.cu = cu;
    p.masks = masks;
    p.out = (bf16*)out;
    p.out_stride = out_stride;
    p.part_o = work;
    p.part_ml = work + 2ll * pl.workers * pl.rows * hd;
    p.uoff = reinterpret_cast<int*>(p.part_ml + 2ll * pl.workers * pl.rows * 2);
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
    p.row_blocks = pl.row_blocks;
    p.zero_tail = zero_tail;
    const int r = pl.rows == 128      ? launch_tile(p, hd, fp8, pl.grid, st)
                  : fp8 && hd == 128 ? launch_tree<true, 128>(p, pl, st)
                  : fp8              ? launch_tree<true, 64>(p, pl, st)
                  : hd == 128        ? launch_tree<false, 128>(p, pl, st)
                                     : launch_tree<false, 64>(p, pl, st);
    if (r || pl.row_blocks) return r;
    if (pl.rows == 128) return hd == 128 ? merge<128, false>(p, pl, zero_tail, st) : merge<64, false>(p, pl, zero_tail, st);
    return hd == 128 ? merge<128, true>(p, pl, zero_tail, st) : merge<64, true>(p, pl, zero_tail, st);
}
