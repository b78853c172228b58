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

constexpr int kEpiSlot = 10;   // the stream workspace of their K splits

typedef int i32x8 __attribute__((ext_vector_type(8)));

// z Phi(z).  erfc(a) e^(a^2) for a = |z| / sqrt(2) is a polynomial in t = 1 / (1 +
// 0.6 a), fitted for the least largest relative error over 0 <= a <= 10.6 (2^-21.6;
// with the roundings 2^-19 down to z = -8 and 2^-17 at -14, where e^(-z^2 / 2) has the
// most of them; a bf16 store's is 2^-8).  A fit of erf alone, of the same absolute
// error, has no bits of the lower tail: Abramowitz and Stegun 7.1.26 was 0.4% off at
// z = -6 and 3.7% at -13.  The exponential is 2^8 of itself, so that it is a normal
// number (the hardware's is 0 below) until nothing of the result is left in bf16; the
// coefficients take that off again, and half of erfc.
__device__ __forceinline__ float gelu_erf(float z) {
    constexpr float s = 0x1p-9f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.42426407f, fabsf(z), 1.0f));
    float c = fmaf(s * -0.0920885652f, t, s * 0.411972642f);
    c = fmaf(c, t, s * -0.64450407f);
    c = fmaf(c, t, s * 0.283816934f);
    c = fmaf(c, t, s * 0.0733853355f);
    c = fmaf(c, t, s * 0.291609466f);
    c = fmaf(c, t, s * 0.337247759f);
    c = fmaf(c, t, s * 0.338560164f) * t * __builtin_amdgcn_exp2f(fmaf(z * z, -0.72134752f, 8.0f));
    return z * (z >= 0.0f ? 1.0f - c : c);   // one less the upper tail, or the lower tail itself
}

// z / (1 + e^-t), the sum 2^-15 of itself: so its reciprocal is a normal number (the
// hardware's is 0 below) as far as t = -97.7, where z = t is the last to leave anything
// in bf16 (less than half of its least step).  The quotient without z is subnormal from
// t = -87.3 on, at most 2^-150 off, and z times that nothing to a bf16 step of 2^-133.
__device__ __forceinline__ float z_sigmoid(float z, float t) {
    return z * (0x1p-15f * __builtin_amdgcn_rcpf(0x1p-15f +
                                                 __builtin_amdgcn_exp2f(fmaf(-1.44269504f, t, -15.0f))));
}

// The activation of R values, its kind looked at once.  (The code is laid out for every
// eight outputs of a tile, 180 KB in all: what two kinds share is there once.)
template <int R>
__device__ __forceinline__ void activate_all(float (&z)[R], int act) {
    if (act == kActNone) return;
    if (act == kActRelu) {
#pragma unroll
        for (int r = 0; r < R; ++r) z[r] = z[r] < 0.0f ? 0.0f : z[r];
    } else if (act == kActGelu) {
#pragma unroll
        for (int r = 0; r < R; ++r) z[r] = gelu_erf(z[r]);
    } else {   // SiLU, or z sigmoid(2 u): the tanh form without its cancellation
        float t[R];
#pragma unroll
        for (int r = 0; r < R; ++r) t[r] = z[r];
        if (act == kActGeluTanh) {
#pragma unroll
            for (int r = 0; r < R; ++r) t[r] = 1.59576912f * z[r] * fmaf(0.044715f * z[r], z[r], 1.0f);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) z[r] = z_sigmoid(z[r], t[r]);
    }
}

// Eight bf16 of a row of Y or R, of the bias, four of the scales: they start at any
// address that an element may have (rows do where N is odd), and global memory
// takes vector accesses there.
typedef uint32_t u32x4_rows __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_rows __attribute__((ext_vector_type(4), aligned(4)));

// What the epilogue of columns n .. n + 7 (n % 8 == 0) takes from memory, loaded
// ahead of the sums: the columns' part, and the token's.
struct EpiCols {
    float ws[8];
    u32x4 bias;
};
struct EpiToken {
    float xs;
    u32x4 r;
};
// Elements n .. n + 7 of a row of N, the last one in the place of those behind it.
__device__ __forceinline__ u32x4 row_end(const uint16_t* row, int n, int N) {
    uint16_t h[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) h[r] = row[min(n + r, N - 1)];
    u32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = h[2 * r] | (static_cast<uint32_t>(h[2 * r + 1]) << 16);
    return v;
}
template <bool F8>
__device__ __forceinline__ EpiCols epi_cols(const EpiParams& p, int n) {
    EpiCols c;
    c.bias = u32x4{0, 0, 0, 0};
    if (n >= p.N) return c;
    if (n + 8 <= p.N) {
        if constexpr (F8) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 w = *reinterpret_cast<const f32x4_rows*>(p.ws + n + 4 * h);
#pragma unroll
                for (int r = 0; r < 4; ++r) c.ws[4 * h + r] = w[r];
            }
        }
        if (p.bias != nullptr) c.bias = *reinterpret_cast<const u32x4_rows*>(p.bias + n);
    } else {   // the row's end: the last column again, so that no load waits for another
        if constexpr (F8) {
#pragma unroll
            for (int r = 0; r < 8; ++r) c.ws[r] = p.ws[min(n + r, p.N - 1)];
        }
        if (p.bias != nullptr) c.bias = row_end(p.bias, n, p.N);
    }
    return c;
}
template <bool F8>
__device__ __forceinline__ EpiToken epi_token(const EpiParams& p, int m, int n) {
    EpiToken t;
    t.r = u32x4{0, 0, 0, 0};
    if (m >= p.M || n >= p.N) return t;
    if constexpr (F8) t.xs = p.xs[m];
    if (p.R == nullptr) return t;
    const uint16_t* at = p.R + static_cast<size_t>(m) * p.N + n;
    if (n + 8 <= p.N) {
        t.r = *reinterpret_cast<const u32x4_rows*>(at);
    } else {
        t.r = row_end(at - n, n, p.N);
    }
    return t;
}

// Columns n .. n + 7 of token m from their sums.
template <bool F8>
__device__ __forceinline__ void epi_store(const EpiParams& p, int m, int n, float (&v)[8],
                                          const EpiCols& c, const EpiToken& t) {
    if (m >= p.M || n >= p.N) return;
    if constexpr (F8) {
        // A sum of codes times the scale of a very large or small token may leave fp32
        // where the weights' scale brings it back: such a scale comes in two parts, the
        // second a power of two after the weights' (1 for any other token).  Nothing is
        // past fp32 on the way then for weights' scales of 2^-124 .. 2^85.  (A branch
        // that took such tokens' scales apart cost 2048 x 14336 x 512 e4m3 37.3 -> 40.8 us,
        // by the length of its code; this 34.5, with the activations' code shared.)
        const bool large = fabsf(t.xs) >= 0x1p80f, small = fabsf(t.xs) <= 0x1p-80f;
        const float xs = t.xs * (large ? 0x1p-64f : small ? 0x1p64f : 1.0f);
        const float after = large ? 0x1p64f : small ? 0x1p-64f : 1.0f;
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = v[r] * xs * c.ws[r] * after;
    }
    if (p.bias != nullptr) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v[2 * r] += __uint_as_float(c.bias[r] << 16);
            v[2 * r + 1] += __uint_as_float(c.bias[r] & 0xffff0000u);
        }
    }
    activate_all(v, p.act);
    if (p.R != nullptr) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v[2 * r] += __uint_as_float(t.r[r] << 16);
            v[2 * r + 1] += __uint_as_float(t.r[r] & 0xffff0000u);
        }
    }
    const u32x4 o = pack_bf16x8(v);
    uint16_t* at = p.Y + static_cast<size_t>(m) * p.N + n;
    if (n + 8 <= p.N) {
        *reinterpret_cast<u32x4_rows*>(at) = o;
    } else {
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (n + r < p.N) at[r] = static_cast<uint16_t>(o[r >> 1] >> (16 * (r & 1)));
    }
}

// The same columns of a K split's fp32 partials [M][N].
__device__ __forceinline__ void epi_store_part(const EpiParams& p, float* part, int m, int n,
                                               const float (&v)[8]) {
    if (m >= p.M || n >= p.N) return;
    float* at = part + static_cast<size_t>(m) * p.N + n;
    if (n + 8 <= p.N) {
        *reinterpret_cast<f32x4_rows*>(at) = f32x4_rows{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_rows*>(at + 4) = f32x4_rows{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (n + r < p.N) at[r] = v[r];
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
// max_splits K splits, whose sums the fp32 partials at `part` carry.  forced: as
// KCMM_GEMM_TILE and KCMM_GEMM_SPLITS say.  Where there is no such plan: 256-token
// tiles without K splits, which any product can run on, of infinite time.
GemmWidePlan gemm_epi_wide_plan(const EpiParams& p, int max_splits, bool forced);
bool gemm_epi_wide(const EpiParams& p, const GemmWidePlan& plan, float* part, uint64_t stream,
                   std::string* err);
// The epilogue of the sum of `splits` fp32 partials [splits][M][N].
bool gemm_epi_sum(const EpiParams& p, const float* part, int splits, uint64_t stream,
                         std::string* err);
}  // namespace dev
}  // namespace kcmm
