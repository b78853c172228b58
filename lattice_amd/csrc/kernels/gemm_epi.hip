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
#include "gemm_epi.hpp"

namespace kcmm {
namespace {

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

// Many tokens: the 256-row tiles, K split where the stream has room for the
// partials (never under a capture: a graph would keep their address).
bool many_tokens(const EpiParams& p, uint64_t stream, std::string* err) {
    dev::GemmWidePlan plan = dev::gemm_epi_wide_plan(p, 8);
    void* part = nullptr;
    if (plan.splits > 1) {
        const size_t bytes = static_cast<size_t>(plan.splits) * p.M * p.N * sizeof(float);
        if (!dev::stream_scratch(stream, 1, bytes)) plan = dev::gemm_epi_wide_plan(p, 1);
        else if (!dev::stream_workspace(stream, 1, bytes, &part, false, err)) return false;
    }
    return dev::gemm_epi_wide(p, plan, static_cast<float*>(part), stream, err);
}

template <bool F8>
bool gemm_epi_typed(const EpiParams& p, uint64_t stream, std::string* err) {
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int forced = dev::tunable_or(dev::Tun::kEpiKernel, 0);
    if (forced == 2 || (forced == 0 && p.M > 64)) return many_tokens(p, stream, err);
    const int cfg = dev::tunable_or(dev::Tun::kEpiCfg, 0);
    switch (cfg) {
        case 114: launch_epi_rows<F8, 1, 1, 4>(p, s); break;
        case 112: launch_epi_rows<F8, 1, 1, 2>(p, s); break;
        case 214: launch_epi_rows<F8, 2, 1, 4>(p, s); break;
        case 212: launch_epi_rows<F8, 2, 1, 2>(p, s); break;
        case 412: launch_epi_rows<F8, 4, 1, 2>(p, s); break;
        case 411: launch_epi_rows<F8, 4, 1, 1>(p, s); break;
        case 122: launch_epi_rows<F8, 1, 2, 2>(p, s); break;
        case 124: launch_epi_rows<F8, 1, 2, 4>(p, s); break;
        case 222: launch_epi_rows<F8, 2, 2, 2>(p, s); break;
        case 221: launch_epi_rows<F8, 2, 2, 1>(p, s); break;
        case 421: launch_epi_rows<F8, 4, 2, 1>(p, s); break;
        case 141: launch_epi_rows<F8, 1, 4, 1>(p, s); break;
        case 142: launch_epi_rows<F8, 1, 4, 2>(p, s); break;
        case 241: launch_epi_rows<F8, 2, 4, 1>(p, s); break;
        case 242: launch_epi_rows<F8, 2, 4, 2>(p, s); break;
        case 441: launch_epi_rows<F8, 4, 4, 1>(p, s); break;
        default:
            if (p.M <= 16) launch_epi_rows<F8, 1, 1, 4>(p, s);
            else if (p.M <= 32) launch_epi_rows<F8, 1, 2, 4>(p, s);
            else launch_epi_rows<F8, 2, 4, 2>(p, s);
    }
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
