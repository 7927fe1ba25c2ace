// The 8-bit paged cache: rows of keys and values quantised while they are written into their slots, and read back as packed
// rows.  Codes are e4m3, [pages][kv head][16][hd] bytes; every (token, kv head) row has one power of two, kept as an exponent
// biased by 127, [pages][kv head][16] bytes:
//
//   2^e = the smallest power of two (from 2^-126) with amax(row) <= 448 * 2^e,   code = e4m3(x * 2^-e), ties to even
//
// A power of two costs no accuracy against amax / 448 (e4m3 is a floating type: its spacing is relative) and makes both
// directions exact up to the one rounding of the code: scaling by it rounds nothing, and code * 2^e has four significant bits,
// which bf16 holds.  A row that holds an infinity or a NaN is stored as exponent 255 with NaN codes; it reads back as NaN.
// Compiled without fast-math (denormal results are kept).
//
// Append: 8191 tokens x 8 heads x 128 in 10.7 us, 4.7 TB/s (the 50 MB would take 7.8).  About 107 instructions per warp and two rows of 128 each of keys and
// values, in 66 % of the issue slots with 81 % of the warps there: between a row's loads and its first code lies the search for its largest
// magnitude.  Two bf16 magnitudes share a word on the way (one at a time: 22 us).  The rows are fetched beside their slot: the two loads'
// latencies do not add up.  Reading back is bound by the memory: 16 x 4096 tokens x 8 heads x 128 in 51 us, 6.0 TB/s (66 us with 16-byte stores).
#include <cuda_fp8.h>

#include "vec.cuh"

namespace {

constexpr int PAGE = 16;
constexpr int THREADS = 256;

__device__ __forceinline__ float pow2(uint32_t biased) {         // 2^(biased - 127); 255 gives infinity
    return __uint_as_float(biased ? biased << 23 : 0x00400000u);
}

struct AppendShape {
    int N, n_kv, hd;
    long long k_stride, v_stride, num_slots;
};

// Eight elements of a row as they lie in memory.
template <typename T>
struct Piece {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void load(const T* src) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(src) + i * 16);
            w[4 * i] = v.x;
            w[4 * i + 1] = v.y;
            w[4 * i + 2] = v.z;
            w[4 * i + 3] = v.w;
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)(2 * sizeof(T)); ++i) w[i] = 0;
    }
    __device__ __forceinline__ uint2 codes(float inv) const {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = __uint_as_float(sizeof(T) == 2 ? w[i] << 16 : w[2 * i % (2 * sizeof(T))]);
            const float hi = __uint_as_float(sizeof(T) == 2 ? w[i] & 0xffff0000u : w[(2 * i + 1) % (2 * sizeof(T))]);
            h[i] = __nv_cvt_float2_to_fp8x2(make_float2(lo * inv, hi * inv), __NV_SATFINITE, __NV_E4M3);
        }
        return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    }
};

// Largest magnitudes of a row of keys and a row of values over LANES lanes, as bits of fp32 (infinities and NaNs are largest).  Two bf16
// magnitudes share a word on the way: half the shuffles.
template <int LANES>
__device__ __forceinline__ uint2 largest(const Piece<bf16>& k, const Piece<bf16>& v) {
    uint32_t a = k.w[0] & 0x7fff7fffu, b = v.w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        a = __vmaxu2(a, k.w[i] & 0x7fff7fffu);
        b = __vmaxu2(b, v.w[i] & 0x7fff7fffu);
    }
    uint32_t m = __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    return make_uint2(m << 16, m & 0xffff0000u);
}
template <int LANES>
__device__ __forceinline__ uint2 largest(const Piece<float>& k, const Piece<float>& v) {
    uint32_t a = 0, b = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a = max(a, k.w[i] & 0x7fffffffu);
        b = max(b, v.w[i] & 0x7fffffffu);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
        b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
    return make_uint2(a, b);
}

// LANES (a power of two, at least hd / 8) lanes share a (token, kv head): its row of keys and its row of values, eight elements of each per
// lane.  (Two of them per lane group: 12.2 us against 10.7 for 8191 tokens, 2.6 against 1.8 for 64.)
template <typename T, int LANES>
__global__ void __launch_bounds__(THREADS)
append_kernel(const T* __restrict__ k, const T* __restrict__ v, const AppendShape s, uint8_t* __restrict__ kc, uint8_t* __restrict__ ke,
              uint8_t* __restrict__ vc, uint8_t* __restrict__ ve, const long long* __restrict__ slots, int* __restrict__ status) {
    kb_dep_trigger();
    kb_dep_wait();
    constexpr int GROUPS = THREADS / LANES;
    const int sub = threadIdx.x % LANES;
    const uint32_t r = blockIdx.x * GROUPS + threadIdx.x / LANES;
    const bool mine = sub * 8 < s.hd;
    Piece<T> x, y;
    x.zero();
    y.zero();
    long long at = -1;
    if (r < (uint32_t)s.N * s.n_kv) {
        const uint32_t n = r / s.n_kv, head = r - n * s.n_kv;
        const long long slot = slots[n];
        if (mine) {                                    // (the rows are fetched beside their slot, not behind it)
            const uint32_t col = head * s.hd + sub * 8;
            x.load(k + n * s.k_stride + col);
            y.load(v + n * s.v_stride + col);
        }
        if (slot >= s.num_slots) {
            if (head == 0 && sub == 0 && status) atomicMax(status, (int)KB_BAD_INDEX);
        } else if (slot >= 0) {
            at = (((unsigned long long)slot / PAGE) * s.n_kv + head) * PAGE + (slot & (PAGE - 1));
        }
    }
    const uint2 m = largest<LANES>(x, y);
    if (at < 0) return;
    // 448 = 1.75 * 2^8: the exponent is that of the magnitude less 8, one more where its mantissa is above 1.75
    const int e = min(max((int)(m.x >> 23) - 8 + ((m.x & 0x7fffffu) > 0x600000u), 1), 254);
    const int f = min(max((int)(m.y >> 23) - 8 + ((m.y & 0x7fffffu) > 0x600000u), 1), 254);
    const bool bad = m.x >= 0x7f800000u, worse = m.y >= 0x7f800000u;
    if (mine) {
        const uint2 c = x.codes(pow2(254 - e)), d = y.codes(pow2(254 - f)), nan = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
        const long long to = at * s.hd + sub * 8;
        *reinterpret_cast<uint2*>(kc + to) = bad ? nan : c;
        *reinterpret_cast<uint2*>(vc + to) = worse ? nan : d;
    }
    if (sub == 0) {
        ke[at] = (uint8_t)(bad ? 255 : e);
        ve[at] = (uint8_t)(worse ? 255 : f);
    }
}

__device__ __forceinline__ void unpack16(const uint4 c, float f, float* x) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> ((i & 1) * 16)), __NV_E4M3);
        const float2 p = __half22float2(__half2(h));
        x[2 * i] = p.x * f;
        x[2 * i + 1] = p.y * f;
    }
}

// Sixteen numbers as whole 32-byte sectors (16-byte stores 32 bytes apart would write each sector in two halves).
__device__ __forceinline__ void store32(void* dst, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                 "r"(w[6]), "r"(w[7])
                 : "memory");
}
__device__ __forceinline__ void store16(bf16* dst, const float* x) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    store32(dst, w);
}
__device__ __forceinline__ void store16(float* dst, const float* x) {
    store32(dst, reinterpret_cast<const uint32_t*>(x));
    store32(dst + 8, reinterpret_cast<const uint32_t*>(x) + 8);
}

struct GatherShape {
    int G, hd, B, max_pages, num_pages, segs, total;
};

// One warp per row (token): its segment and page are looked up once, then the lanes walk the row's 2 * G * hd / 16 pieces of
// sixteen codes.
template <typename T>
__global__ void __launch_bounds__(THREADS)
gather_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ ke, const uint8_t* __restrict__ vc, const uint8_t* __restrict__ ve,
              const GatherShape s, const int* __restrict__ table, const int* __restrict__ seq, const int* __restrict__ first,
              const int* __restrict__ cu, T* __restrict__ k, T* __restrict__ v, int* __restrict__ status) {
    kb_dep_trigger();
    kb_dep_wait();
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    if (row >= s.total) return;
    int lo = 0, hi = s.segs;                             // the segment with cu[lo] <= row < cu[lo + 1]
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (cu[m] <= row) lo = m; else hi = m;
    }
    const int p = first[lo] + (int)row - cu[lo], b = seq[lo], pi = p / PAGE;
    const int page = b >= 0 && b < s.B && p >= 0 && pi < s.max_pages ? table[(long long)b * s.max_pages + pi] : -1;
    const bool ok = page >= 0 && page < s.num_pages;
    if (!ok && lane == 0 && status) atomicMax(status, (int)KB_BAD_INDEX);
    const int per = s.hd >> 4, pieces = s.G * per;
    for (int c0 = 0; c0 < 2 * pieces; c0 += 128) {
        uint4 w[4];
        uint32_t e[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c = c0 + u * 32 + lane;
            w[u] = make_uint4(0, 0, 0, 0);
            e[u] = 127;
            if (ok && c < 2 * pieces) {
                const bool isv = c >= pieces;
                const int d = isv ? c - pieces : c, g = d / per;
                const long long at = ((long long)page * s.G + g) * PAGE + p % PAGE;
                w[u] = *reinterpret_cast<const uint4*>((isv ? vc : kc) + at * s.hd + (d % per) * 16);
                e[u] = (isv ? ve : ke)[at];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c = c0 + u * 32 + lane;
            if (c < 2 * pieces) {
                const bool isv = c >= pieces;
                float x[16];
                unpack16(w[u], pow2(e[u]), x);
                T* dst = (isv ? v : k) + row * s.G * s.hd + (long long)(isv ? c - pieces : c) * 16;
                store16(dst, x);
            }
        }
    }
}

template <typename T, int LANES>
int launch_append(const void* k, const void* v, const AppendShape& s, void* kc, void* ke, void* vc, void* ve, const long long* slots,
                  int* status, cudaStream_t st) {
    const long long rows = (long long)s.N * s.n_kv, groups = THREADS / LANES;
    if (rows > 0x7fffffffll - groups) return 5;
    return kb_launch_dep(append_kernel<T, LANES>, dim3((unsigned)((rows + groups - 1) / groups)), dim3(THREADS), 0, st, (const T*)k, (const T*)v, s,
                         (uint8_t*)kc, (uint8_t*)ke, (uint8_t*)vc, (uint8_t*)ve, slots, status);
}

template <typename T>
int append_by_lanes(const void* k, const void* v, const AppendShape& s, void* kc, void* ke, void* vc, void* ve, const long long* slots,
                    int* status, cudaStream_t st) {
    if (s.hd <= 64) return launch_append<T, 8>(k, v, s, kc, ke, vc, ve, slots, status, st);
    if (s.hd <= 128) return launch_append<T, 16>(k, v, s, kc, ke, vc, ve, slots, status, st);
    return launch_append<T, 32>(k, v, s, kc, ke, vc, ve, slots, status, st);
}

}  // namespace

// k, v: [N, n_kv * hd] rows (type 0 = bf16, 1 = fp32) with the given strides; slots as in kb_kv_append: negative ones are skipped,
// one at or past num_slots is recorded as KB_BAD_INDEX and skipped.  hd: a multiple of 16, at most 256.
KB_API int kb_kv_append_fp8(const void* k, const void* v, long long k_stride, long long v_stride, void* kc, void* ke, void* vc, void* ve,
                            const long long* slots, int N, int n_kv, int hd, long long num_slots, int type, int* status, cudaStream_t st) {
    const int piece = type == 0 ? 8 : 4;                 // elements of a 16-byte access
    if (N < 1 || n_kv < 1 || hd < 16 || hd > 256 || hd % 16 || k_stride % piece || v_stride % piece || num_slots < 0 || type < 0 || type > 1 ||
        ((uintptr_t)k | (uintptr_t)v | (uintptr_t)kc | (uintptr_t)vc) % 16)
        return 5;
    const AppendShape s{N, n_kv, hd, k_stride, v_stride, num_slots};
    if (type == 0) return append_by_lanes<bf16>(k, v, s, kc, ke, vc, ve, slots, status, st);
    return append_by_lanes<float>(k, v, s, kc, ke, vc, ve, slots, status, st);
}

// k, v: [total, G, hd] packed rows (type 0 = bf16, 1 = fp32); segments as in kb_kv_gather.  Rows whose page is out of range are zero and
// recorded as KB_BAD_INDEX.
KB_API int kb_kv_gather_fp8(const void* kc, const void* ke, const void* vc, const void* ve, int G, int hd, const int* table, int B, int max_pages,
                            int num_pages, const int* seq, const int* first, const int* cu, int segs, void* k, void* v, int total, int type,
                            int* status, cudaStream_t st) {
    if (G < 1 || hd < 16 || hd > 256 || hd % 16 || B < 1 || segs < 1 || total < 1 || type < 0 || type > 1 ||
        ((uintptr_t)k | (uintptr_t)v) % 32 || ((uintptr_t)kc | (uintptr_t)vc) % 16)
        return 5;
    const GatherShape s{G, hd, B, max_pages, num_pages, segs, total};
    const unsigned blocks = (unsigned)((total + THREADS / 32 - 1) / (THREADS / 32));
    if (type == 0)
        return kb_launch_dep(gather_kernel<bf16>, dim3(blocks), dim3(THREADS), 0, st, (const uint8_t*)kc, (const uint8_t*)ke, (const uint8_t*)vc,
                             (const uint8_t*)ve, s, table, seq, first, cu, (bf16*)k, (bf16*)v, status);
    return kb_launch_dep(gather_kernel<float>, dim3(blocks), dim3(THREADS), 0, st, (const uint8_t*)kc, (const uint8_t*)ke, (const uint8_t*)vc,
                         (const uint8_t*)ve, s, table, seq, first, cu, (float*)k, (float*)v, status);
}
