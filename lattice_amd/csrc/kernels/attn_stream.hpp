// Pieces of the kernels that stream K/V pages through registers (attn_decode.hip,
// attn_shared.hip): a 32-token tile's loads, their turn into MFMA operand
// layout, V^T by selection products.
#pragma once
#include <cmath>

#include "common.hpp"

namespace kcmm {
namespace {

__device__ __forceinline__ float wave_max_across_groups(float x) {
    // lanes j, j+16, j+32, j+48 hold the same column; combine them.
    x = fmaxf(x, __shfl_xor(x, 16));
    x = fmaxf(x, __shfl_xor(x, 32));
    return x;
}

__device__ __forceinline__ float wave_sum_across_groups(float x) {
    x += __shfl_xor(x, 16);
    x += __shfl_xor(x, 32);
    return x;
}

template <int DT>
__device__ __forceinline__ f32x4 mfma16x16x32(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == kDtF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                       0);
}

// One 32-token tile: 2 halves of 16 tokens, KC 16-byte fragments per lane
// each; after fix_lines, k[h][kc] of lane (ln, lg) holds bytes
// (4kc + lg)*16 .. +16 of token 16h + ln's head row (the MFMA A layout).
template <int KC>
struct Tile {
    u32x4 k[2][KC];
    u32x4 v[2][KC];
};

// Row rotation by 8 inside each 16-lane row (DPP row_ror:8; its own inverse).
__device__ __forceinline__ uint32_t ror8(uint32_t x) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x128, 0xF, 0xF, false));
}

// x was loaded as: lane (r, lg) <- token (r & 7), bytes (4*(r >> 3) + lg)*16
// of a 128-byte line; y the same for tokens 8..15.  Afterwards x holds the
// first 64 bytes of tokens 0..15 and y the second 64 bytes, lane r = token r.
__device__ __forceinline__ void fix_lines(u32x4& x, u32x4& y, bool low8) {
    u32x4 nx, ny;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t rx = ror8(x[c]);
        const uint32_t ry = ror8(y[c]);
        nx[c] = low8 ? x[c] : ry;
        ny[c] = low8 ? rx : y[c];
    }
    x = nx;
    y = ny;
}

__device__ __forceinline__ u32x4 load_stream(const uint8_t* a) {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a));
}

// B operand of a 16x16x32 MFMA that selects 16 consecutive k indices:
// E[k][j] = (k == 16*sub + j).  Multiplying an A operand by it returns the
// selected A columns in C layout, i.e. transposed relative to the A layout.
template <int DT>
__device__ __forceinline__ u32x4 select_operand(int sub, int ln, int lg) {
    constexpr uint32_t one = DT == kDtF16 ? 0x3C00u : 0x3F80u;
    u32x4 e = u32x4{0, 0, 0, 0};
    const int k = 16 * sub + ln;          // the k that column ln selects
    if ((k >> 3) == lg) {
        const int t = k & 7;              // item within the lane's 8 k values
        e[t >> 1] = (t & 1) ? (one << 16) : one;
    }
    return e;
}

// Two fp32 values that hold exactly representable 16-bit values -> packed pair.
template <int DT>
__device__ __forceinline__ uint32_t pack_exact(float lo, float hi) {
    if constexpr (DT == kDtF16) {
        return f32_to_f16_bits(lo) | (f32_to_f16_bits(hi) << 16);
    } else {
        return (__float_as_uint(lo) >> 16) | (__float_as_uint(hi) & 0xffff0000u);
    }
}

// Eight e4m3 values (two dwords) -> eight bf16, exactly (every e4m3 value
// is a bf16 value); the page scale is applied outside, in fp32.
__device__ __forceinline__ u32x4 fp8x8_to_bf16(uint32_t d0, uint32_t d1) {
    u32x4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d0, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d0, 1.0f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d1, 1.0f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d1, 1.0f, true));
    return r;
}

// First of the four consecutive dims that lane group lg holds in acc[db]
// (rows 4lg .. 4lg+3 of the O^T block).
template <bool F8>
__device__ __forceinline__ int dim_offset(int db, int lg) {
    if constexpr (F8) {
        const int kc = db >> 1, sub = db & 1;
        return (kc >> 1) * 64 + (kc & 1) * 8 + 32 * sub + 4 * lg + (lg >= 2 ? 8 : 0);
    } else {
        return 16 * db + 4 * lg;
    }
}

}  // namespace
}  // namespace kcmm
