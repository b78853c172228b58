// Products with bias, activation and residual in their epilogue, Y[M][N] =
// bf16(act(X W^T (* xscale[m] * wscale[n]) + bias[n]) + residual[m][n]): bf16
// operands, or e4m3 codes with an fp32 scale per token and per weight row on
// the fp8 matrix instructions (twice the bf16 rate).  The sums, the scales, the
// activation and the addition are fp32; the store rounds once.  One thing less
// than fp32 is the instruction's own: it adds the products of 8 consecutive k
// aligned to the largest and drops what lies below 2^-13 of that one (measured;
// the sums of 8 and the accumulator are fp32).  With rows quantised as here the
// outputs' error against 64 bits stays that of the bf16 store (1.7e-3 of the
// norm with and without), a 40th of the operands' own rounding to 2^-4.
//
// gemm_epi_rows: one workgroup of 8 waves on 16 NB weight rows x 16 MB tokens,
// K split over its waves, the sums joined in LDS in wave order: no partials in
// memory and no second launch, so a captured call needs no workspace.
//  * both operands go from memory to registers in the layout of the matrix
//    instructions: lane (row ln, group lg) takes 32 bytes at 32 lg of a
//    128-byte line of its row.  The instructions sum over k in whatever order
//    both operands have in common, so no operand is permuted;
//  * stage s + 1 (U lines of each row a wave, whole lines) is in flight while
//    stage s is consumed.
#include <algorithm>
#include <type_traits>

#include "../device_api.hpp"
#include "common.hpp"

namespace kcmm {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

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

constexpr int kRowWaves = 8;

template <bool F8, int NB, int MB, int U, bool VEC>
__global__ __launch_bounds__(64 * kRowWaves) void gemm_epi_rows(EpiParams p) {
    __shared__ f32x4 red[kRowWaves][NB * MB][64];
    const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16 * NB, m0 = blockIdx.y * 16 * MB;
    const int lines = static_cast<int>((p.kb + 127) / 128);            // the last may be partial
    const int full = static_cast<int>(p.kb / (128 * kRowWaves * U));   // stages of whole lines

    // rows past the last are clamped; their outputs are not stored
    const uint8_t* wr[NB];
    const uint8_t* xr[MB];
#pragma unroll
    for (int i = 0; i < NB; ++i) wr[i] = p.W + static_cast<size_t>(min(n0 + 16 * i + ln, p.N - 1)) * p.kb;
#pragma unroll
    for (int j = 0; j < MB; ++j) xr[j] = p.X + static_cast<size_t>(min(m0 + 16 * j + ln, p.M - 1)) * p.kb;

    f32x4 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    struct Stage {
        u32x4 a[U][NB][2], b[U][MB][2];
    };
    // Stage s < full: U consecutive lines of each wave.  Stage `full`: what is
    // left, a line a wave in turn, addresses held inside the row.
    auto load = [&](Stage& t, int s) {
        uint32_t o[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (s < full) o[u][h] = ((s * kRowWaves + wave) * U + u) * 128 + lg * 32 + h * 16;
                else o[u][h] = min((full * kRowWaves * U + wave + kRowWaves * u) * 128 + lg * 32 + h * 16,
                                   p.kb - 16);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < MB; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) t.b[u][j][h] = *reinterpret_cast<const u32x4*>(xr[j] + o[u][h]);
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    t.a[u][i][h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wr[i] + o[u][h]));
        }
    };
    auto compute = [&](Stage& t, int s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s == full) {
                const int line = full * kRowWaves * U + wave + kRowWaves * u;
                if (line >= lines) continue;
                if (line * 128 + 128 > static_cast<int>(p.kb)) {   // the row's end: zeros behind it
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (line * 128 + lg * 32 + h * 16 < static_cast<int>(p.kb)) continue;
#pragma unroll
                        for (int i = 0; i < NB; ++i) t.a[u][i][h] = u32x4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < MB; ++j) t.b[u][j][h] = u32x4{0, 0, 0, 0};
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int j = 0; j < MB; ++j) acc[i][j] = mfma_line<F8>(t.a[u][i], t.b[u][j], acc[i][j]);
        }
    };
    const int stages = full + (lines > full * kRowWaves * U);
    Stage t0, t1;
    load(t0, 0);
    int s = 0;
    for (; s + 2 < stages; s += 2) {
        load(t1, s + 1);
        compute(t0, s);
        load(t0, s + 2);
        compute(t1, s + 1);
    }
    if (s + 1 < stages) {
        load(t1, s + 1);
        compute(t0, s);
        compute(t1, s + 1);
    } else {
        compute(t0, s);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) red[wave][i * MB + j][lane] = acc[i][j];
    __syncthreads();
    // block b: weight rows 16 (b / MB) + 4 lg .. + 3, token 16 (b % MB) + ln
    for (int b = wave; b < NB * MB; b += kRowWaves) {
        f32x4 v = red[0][b][lane];
#pragma unroll
        for (int w = 1; w < kRowWaves; ++w) v += red[w][b][lane];
        epi_store4<F8, VEC>(p, m0 + 16 * (b % MB) + ln, n0 + 16 * (b / MB) + 4 * lg, v);
    }
}

template <bool F8, int NB, int MB, int U>
void launch_epi_rows(const EpiParams& p, hipStream_t s) {
    const dim3 grid((p.N + 16 * NB - 1) / (16 * NB), (p.M + 16 * MB - 1) / (16 * MB));
    if (p.N % 4 == 0)
        hipLaunchKernelGGL((gemm_epi_rows<F8, NB, MB, U, true>), grid, dim3(64 * kRowWaves), 0, s, p);
    else
        hipLaunchKernelGGL((gemm_epi_rows<F8, NB, MB, U, false>), grid, dim3(64 * kRowWaves), 0, s, p);
}

template <bool F8>
bool gemm_epi_typed(const EpiParams& p, uint64_t stream, std::string* err) {
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (p.M <= 16) launch_epi_rows<F8, 1, 1, 4>(p, s);
    else if (p.M <= 32) launch_epi_rows<F8, 1, 2, 4>(p, s);
    else launch_epi_rows<F8, 2, 4, 2>(p, s);
    KCMM_HIP_CHECK(hipGetLastError(), err);
    return true;
}

}  // namespace

namespace dev {

bool gemm_epi(const GemmEpiArgs& a, std::string* err) {
    EpiParams p{};
    p.X = reinterpret_cast<const uint8_t*>(a.x);
    p.W = reinterpret_cast<const uint8_t*>(a.w);
    p.xs = reinterpret_cast<const float*>(a.xscale);
    p.ws = reinterpret_cast<const float*>(a.wscale);
    p.bias = reinterpret_cast<const uint16_t*>(a.bias);
    p.R = reinterpret_cast<const uint16_t*>(a.residual);
    p.Y = reinterpret_cast<uint16_t*>(a.y);
    p.M = static_cast<int>(a.m);
    p.N = static_cast<int>(a.n);
    p.act = a.act;
    const bool f8 = a.xscale != 0;
    p.kb = a.k * (f8 ? 1 : 2);
    return f8 ? gemm_epi_typed<true>(p, a.stream, err) : gemm_epi_typed<false>(p, a.stream, err);
}

}  // namespace dev
}  // namespace kcmm
