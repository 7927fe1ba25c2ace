// 4-bit weights as Int4Weight lays them out: what both product kernels share.
#pragma once
#include "common.cuh"

namespace codes4 {

constexpr int KB = 64;                                 // inputs of a block: 512 contiguous bytes, 16 rows x 64 inputs

struct Shape {
    int M, N, K, nt, kb, ng;                           // tokens, rows, inputs; row tiles of 16, blocks of 64 inputs, groups
    long long x_stride, y_stride, c_stride;
};

// One word (eight codes) -> four pairs of bf16: (row r, inputs 0 1), (r + 8, 0 1), (r, 2 3), (r + 8, 2 3).  Masked alone, a
// nibble in the low byte of a half word is a subnormal bf16 number: code * 2^-133 (bits 0 - 3) or code * 2^-129 (bits 4 - 7, of which the top one
// is the exponent's lowest: it counts the same).  Times 2^127 less 8 units that is (code - 8) / 64 for row r and (code - 8) / 4 for row r + 8, exactly.
constexpr float UNIT0 = 64.f, UNIT1 = 4.f;
__device__ __forceinline__ void expand(uint32_t w, uint32_t* a) {
    const __nv_bfloat162 up = __float2bfloat162_rn(1.70141183460469231732e38f), o0 = __float2bfloat162_rn(-0.125f), o1 = __float2bfloat162_rn(-2.f);
    const uint32_t z = w >> 8, v[4] = {w & 0x000f000fu, w & 0x00f000f0u, z & 0x000f000fu, z & 0x00f000f0u};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 d = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v[i]), up, i & 1 ? o1 : o0);
        a[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
}

// Products of more than 16 tokens (gemm_int4_tile_sm100.cu).
int launch_tile(const __nv_bfloat16* x, const uint4* packed, const __nv_bfloat16* scales, const __nv_bfloat16* c, __nv_bfloat16* y, const Shape& s,
                int group, int sms, int* status, cudaStream_t st);

}  // namespace codes4
