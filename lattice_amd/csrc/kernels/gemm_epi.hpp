// What the epilogue products share (gemm_epi.hip, gemm_epi_wide.hip): operands,
// the matrix instruction on a 128-byte line of both, and the epilogue.
#pragma once
#include "../device_api.hpp"
#include "common.hpp"

namespace kcmm {

struct EpiParams {
    const uint8_t* X;        // [M][K], bf16 or e4m3
    const uint8_t* W;        // [N][K]
    const float* xs;         // [M]; e4m3 only
    const float* ws;         // [N]
    const uint16_t* bias;    // [N] or null
    const uint16_t* R;       // [M][N] or null (may be Y)
    uint16_t* Y;             // [M][N]
    int M, N;
    uint32_t kb;             // bytes of an operand's row (a multiple of 16)
    int act;
};

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// erfc(a) e^(a^2) for a >= 0 as a polynomial in t = 1 / (1 + 0.3275911 a)
// (Abramowitz and Stegun 7.1.26): erfc is off by at most 1.5e-7, a bf16
// rounding of the activation by 2^-9 of it.
__device__ __forceinline__ float gelu_erf(float z) {
    const float a = fabsf(z) * 0.70710678f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, a, 1.0f));
    float c = fmaf(1.061405429f, t, -1.453152027f);
    c = fmaf(c, t, 1.421413741f);
    c = fmaf(c, t, -0.284496736f);
    c = fmaf(c, t, 0.254829592f) * t * __expf(-a * a);
    // z Phi(z): one less the upper tail, or the lower tail itself
    return z * (z >= 0.0f ? fmaf(-0.5f, c, 1.0f) : 0.5f * c);
}

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case kActRelu: return z < 0.0f ? 0.0f : z;
        case kActGelu: return gelu_erf(z);
        case kActGeluTanh:   // z sigmoid(2 u): the tanh form without its cancellation
            return z / (1.0f + __expf(-1.59576912f * z * fmaf(0.044715f * z, z, 1.0f)));
        case kActSilu: return z / (1.0f + __expf(-z));
        default: return z;
    }
}

// The activation of R values, its kind looked at once.
template <int R>
__device__ __forceinline__ void activate_all(float (&z)[R], int act) {
    switch (act) {
#define KCMM_ACT_CASE(A)                                          \
    case A:                                                       \
        _Pragma("unroll") for (int r = 0; r < R; ++r) z[r] = activate(z[r], A); \
        break;
        KCMM_ACT_CASE(kActRelu)
        KCMM_ACT_CASE(kActGelu)
        KCMM_ACT_CASE(kActGeluTanh)
        KCMM_ACT_CASE(kActSilu)
#undef KCMM_ACT_CASE
        default: break;
    }
}

// Outputs (m, n .. n + 3) from their sums.  VEC: N % 4 == 0.
template <bool F8, bool VEC>
__device__ __forceinline__ void epi_store4(const EpiParams& p, int m, int n, f32x4 v) {
    if (m >= p.M || n >= p.N) return;
    if constexpr (F8) v *= p.xs[m];
    const size_t at = static_cast<size_t>(m) * p.N + n;
    if constexpr (VEC) {
        if constexpr (F8) v *= *reinterpret_cast<const f32x4*>(p.ws + n);
        if (p.bias != nullptr) {
            const u32x2 b = *reinterpret_cast<const u32x2*>(p.bias + n);
            v += f32x4{__uint_as_float(b[0] << 16), __uint_as_float(b[0] & 0xffff0000u),
                       __uint_as_float(b[1] << 16), __uint_as_float(b[1] & 0xffff0000u)};
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = activate(v[r], p.act);
        if (p.R != nullptr) {
            const u32x2 b = *reinterpret_cast<const u32x2*>(p.R + at);
            v += f32x4{__uint_as_float(b[0] << 16), __uint_as_float(b[0] & 0xffff0000u),
                       __uint_as_float(b[1] << 16), __uint_as_float(b[1] & 0xffff0000u)};
        }
        u32x2 o;
        o[0] = f32_to_bf16_bits(v[0]) | (f32_to_bf16_bits(v[1]) << 16);
        o[1] = f32_to_bf16_bits(v[2]) | (f32_to_bf16_bits(v[3]) << 16);
        *reinterpret_cast<u32x2*>(p.Y + at) = o;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (n + r >= p.N) continue;
            float z = v[r];
            if constexpr (F8) z *= p.ws[n + r];
            if (p.bias != nullptr) z += bf16_bits_to_f32(p.bias[n + r]);
            z = activate(z, p.act);
            if (p.R != nullptr) z += bf16_bits_to_f32(p.R[at + r]);
            p.Y[at + r] = static_cast<uint16_t>(f32_to_bf16_bits(z));
        }
    }
}

// 16 x 16 outputs += 128 bytes of k: lane (ln, lg) holds 32 bytes of row ln.
template <bool F8>
__device__ __forceinline__ f32x4 mfma_line(const u32x4 (&a)[2], const u32x4 (&b)[2], f32x4 c) {
    if constexpr (F8) {
        const i32x8 av = __builtin_bit_cast(i32x8, __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7));
        const i32x8 bv = __builtin_bit_cast(i32x8, __builtin_shufflevector(b[0], b[1], 0, 1, 2, 3, 4, 5, 6, 7));
        // formats 0, 0: e4m3; block scales of constant 0: the form without them
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 0, 0, 0, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[0]),
                                                    __builtin_bit_cast(bf16x8, b[0]), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[1]),
                                                       __builtin_bit_cast(bf16x8, b[1]), c, 0, 0, 0);
    }
}

}  // namespace

namespace dev {
// The product on 256-row tiles (gemm_epi_wide.hip) and the plan for it; at most
// max_splits K splits, whose sums the fp32 partials at `part` carry.
GemmWidePlan gemm_epi_wide_plan(const EpiParams& p, int max_splits);
bool gemm_epi_wide(const EpiParams& p, const GemmWidePlan& plan, float* part, uint64_t stream,
                   std::string* err);
}  // namespace dev
}  // namespace kcmm
