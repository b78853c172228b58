// The epilogue products (gemm_epi.hip) for prompt-sized token counts: the tiles,
// waves and LDS ring of gemm_wide.hip on 128-byte lines of either type.  A line
// is 64 bf16 (two matrix instructions of 16 cycles a block) or 128 e4m3 (one of
// 32 cycles), so a chunk costs the same bytes, LDS cycles and matrix cycles for
// both, and e4m3 does twice the work in them.
//  * any N and M: rows past the end are clamped, their outputs not stored;
//  * K of any number of 16-byte pieces: the last line's loads are held inside
//    the row, and both operands' pieces behind its end are zeroed on their way
//    from LDS (one operand would not do: what lies there may be NaN);
//  * the epilogue runs on the accumulators, 8 consecutive columns a lane; with K
//    splits the sums go through fp32 partials, and a second kernel adds them in
//    split order and runs it.
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "../device_api.hpp"
#include "common.hpp"
#include "gemm_epi.hpp"
#include "wide_pipe.hpp"

namespace kcmm {
namespace {

struct EpiWideParams {
    EpiParams e;
    float* part;         // non-null: fp32 partials [split][M][N]
    int lines;           // 128-byte lines of each K split (the last one's last may be partial)
    // the grid's x range, as in gemm_wide.hip
    int nw[2], full[2], fb[2], rag[2];
};

constexpr int kEpiWideLds = 160 * 1024;

// One tile: 256 weight rows of weight tile tn by BM = 64 * FB tokens from m0.
// The phases, waits and places are those of wide_tile in gemm_wide.hip.
template <bool F8, int FB, bool WNT>
__device__ __forceinline__ void epi_wide_tile(const EpiWideParams& p, uint8_t* lds, int tn, int m0) {
    constexpr int BM = 64 * FB;
    constexpr int WT = 256 * 128, XT = BM * 128;   // bytes of a line's W and X tiles
    static_assert(2 * WT + 3 * XT <= kEpiWideLds, "LDS");
    const EpiParams& e = p.e;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ln = lane & 15, lg = lane >> 4;
    const int wn = wave & 3, wm = wave >> 2;
    const int n0 = tn * 256;
    const uint32_t rowb = e.kb;
    const uint32_t kbeg = blockIdx.y * p.lines * 128u;
    const int nlines = min(p.lines, static_cast<int>((rowb - kbeg + 127) / 128));
    // bytes of the last line; less than 128: its loads end with the row
    const int last = static_cast<int>(min(rowb - kbeg, static_cast<uint32_t>(nlines) * 128u)) -
                     (nlines - 1) * 128;

    const int lrow = lane >> 3;
    const int wpiece = (lane & 7) ^ ((lrow & 3) | ((wave & 1) << 2));
    const int xpiece = (lane & 7) ^ lrow;
    const uint32_t wback = max(0, wpiece * 16 - (last - 16)), xback = max(0, xpiece * 16 - (last - 16));
    uint32_t wof[4], xof[FB];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        wof[i] = static_cast<uint32_t>(min(n0 + 8 * (8 * i + wave) + lrow, e.N - 1)) * rowb + wpiece * 16;
#pragma unroll
    for (int i = 0; i < FB; ++i)
        xof[i] = static_cast<uint32_t>(min(m0 + 8 * (8 * i + wave) + lrow, e.M - 1)) * rowb + xpiece * 16;
    const uint8_t* wk = e.W + kbeg;
    const uint8_t* xk = e.X + kbeg;
    auto issue_w = [&](int c, int slot) {
        uint8_t* dst = lds + slot * WT + wave * 1024;
        const uint8_t* src = wk + static_cast<size_t>(c) * 128;
        const uint32_t back = c + 1 == nlines ? wback : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (WNT) load_lds16_nt(src + (wof[i] - back), dst + i * 8192);
            else load_lds16(src + (wof[i] - back), dst + i * 8192);
        }
    };
    auto issue_x = [&](int c, int slot) {
        uint8_t* dst = lds + 2 * WT + slot * XT + wave * 1024;
        const uint8_t* src = xk + static_cast<size_t>(c) * 128;
        const uint32_t back = c + 1 == nlines ? xback : 0;
#pragma unroll
        for (int i = 0; i < FB; ++i) load_lds16(src + (xof[i] - back), dst + i * 8192);
    };

    f32x4 acc[2][2][2][FB];   // [weight half][block][token half][block]
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < FB; ++j) acc[a][i][b][j] = f32x4{0, 0, 0, 0};

    const int a_lane = (wn * 32 + 8 * (ln >> 2) + (ln & 3)) * 128;
    const int b_lane = 2 * WT + (wm * 16 * FB + ln) * 128;
    const int sw0 = ((0 + lg) ^ (ln & 7)) * 16, sw1 = ((4 + lg) ^ (ln & 7)) * 16;
    u32x4 a[2][2][2], b[FB][2];   // [half][block][piece lg, piece 4 + lg], [block][piece]
    auto read_a = [&](int c) {
        const uint8_t* st = lds + (c & 1) * WT + a_lane;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[h][i][0] = *reinterpret_cast<const u32x4*>(st + sw0 + h * 16384 + i * 512);
                a[h][i][1] = *reinterpret_cast<const u32x4*>(st + sw1 + h * 16384 + i * 512);
            }
    };
    auto read_b = [&](int h, int slot) {
        const uint8_t* st = lds + slot * XT + b_lane + h * (XT / 2);
#pragma unroll
        for (int j = 0; j < FB; ++j) {
            b[j][0] = *reinterpret_cast<const u32x4*>(st + sw0 + j * 2048);
            b[j][1] = *reinterpret_cast<const u32x4*>(st + sw1 + j * 2048);
        }
    };
    // the last line's pieces behind the row's end
    const bool cut[2] = {lg * 16 >= last, (4 + lg) * 16 >= last};
    auto cut_a = [&]() {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (cut[k]) a[h][i][k] = u32x4{0, 0, 0, 0};
    };
    auto cut_b = [&]() {
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (cut[k]) b[j][k] = u32x4{0, 0, 0, 0};
    };
    auto mfmas = [&](int bh) {
        if constexpr (F8) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < FB; ++j)
                        acc[h][i][bh][j] = mfma_line<true>(a[h][i], b[j], acc[h][i][bh][j]);
        } else {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < FB; ++j)
                            acc[h][i][bh][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                __builtin_bit_cast(bf16x8, a[h][i][ks]),
                                __builtin_bit_cast(bf16x8, b[j][ks]), acc[h][i][bh][j], 0, 0, 0);
        }
    };
    int sx = 0;   // X slot of line c (c % 3)
    auto line = [&](int c, auto steady_tag) {
        constexpr bool ST = decltype(steady_tag)::value;
        const int sn = sx == 0 ? 2 : sx - 1;   // slot of line c + 2
        const bool ends = !ST && c + 1 == nlines && last < 128;
        read_b(0, sx);
        read_a(c);
        if constexpr (ST) issue_x(c + 2, sn);
        wait_vm_lgkm0<63>();   // the fragments only
        if (ends) {
            cut_a();
            cut_b();
        }
        phase_barrier();
        __builtin_amdgcn_s_setprio(1);
        mfmas(0);
        __builtin_amdgcn_s_setprio(0);
        phase_barrier();
        read_b(1, sx);
        if constexpr (ST) issue_w(c + 2, c & 1);
        wait_vm_lgkm0<ST ? FB + 4 : 0>();
        if (ends) cut_b();
        phase_barrier();
        __builtin_amdgcn_s_setprio(1);
        mfmas(1);
        __builtin_amdgcn_s_setprio(0);
        phase_barrier();
        sx = sx == 2 ? 0 : sx + 1;
    };

    const int second = min(1, nlines - 1);   // (a single line twice: nothing reads the second)
    issue_x(0, 0);
    issue_w(0, 0);
    issue_x(second, 1);
    issue_w(second, 1);
    wait_vm_lgkm0<FB + 4>();
    phase_barrier();
    if (wm == 1) phase_barrier();   // half a phase behind
    int c = 0;
    for (; c < nlines - 2; ++c) line(c, std::true_type{});
    for (; c < nlines; ++c) line(c, std::false_type{});
    if (wm == 0) phase_barrier();

    // acc[ah][i][bh][j][r] = token m0 + bh*BM/2 + wm*16*FB + 16j + ln, weight
    // row (of half ah) wn*32 + 8*lg + 4*i + r
    auto token = [&](int bh, int j) { return m0 + bh * (BM / 2) + wm * 16 * FB + 16 * j + ln; };
    const bool plain = p.part == nullptr;
#pragma unroll
    for (int ah = 0; ah < 2; ++ah) {
        const int n = n0 + ah * 128 + wn * 32 + 8 * lg;
        const EpiCols cols = epi_cols<F8>(e, plain ? n : e.N);
#pragma unroll
        for (int bh = 0; bh < 2; ++bh) {
            EpiToken t[FB];   // every load of the half before its stores
#pragma unroll
            for (int j = 0; j < FB; ++j) t[j] = epi_token<F8>(e, plain ? token(bh, j) : e.M, n);
#pragma unroll
            for (int j = 0; j < FB; ++j) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[4 * i + r] = acc[ah][i][bh][j][r];
                if (plain) epi_store<F8>(e, token(bh, j), n, v, cols, t[j]);
                else epi_store_part(e, p.part + static_cast<size_t>(blockIdx.y) * e.M * e.N, token(bh, j), n, v);
            }
        }
    }
}

template <bool F8, bool WNT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void gemm_epi_wide_kernel(EpiWideParams p) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kEpiWideLds];
    int i = blockIdx.x, fb = 0, tn = 0, m0 = 0;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        const int n = p.nw[z] * p.full[z];
        if (fb == 0 && i < n) {
            // blocks of 8 token tiles, token tiles fastest
            const int t = xcd_order(i, n);
            const int mg = t / (8 * p.nw[z]), rem = t - mg * 8 * p.nw[z];
            const int gm = min(8, p.full[z] - mg * 8);
            tn = rem / gm;
            m0 = (mg * 8 + rem - tn * gm) * 64 * p.fb[z];
            fb = p.fb[z];
            if (z) tn += p.nw[0];
        }
        i -= n;
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        const int n = p.rag[z] > 0 ? p.nw[z] : 0;
        if (fb == 0 && i < n) {
            tn = xcd_order(i, n) + (z ? p.nw[0] : 0);
            m0 = p.full[z] * 64 * p.fb[z];
            fb = p.rag[z];
        }
        i -= n;
    }
    switch (fb) {
        case 1: epi_wide_tile<F8, 1, WNT>(p, lds, tn, m0); break;
        case 2: epi_wide_tile<F8, 2, WNT>(p, lds, tn, m0); break;
        case 3: epi_wide_tile<F8, 3, WNT>(p, lds, tn, m0); break;
        case 4: epi_wide_tile<F8, 4, WNT>(p, lds, tn, m0); break;
        default: break;
    }
}

// The epilogue of the summed K splits, 8 columns a thread.
template <bool F8>
__global__ __launch_bounds__(256) void sum_partials_epi(EpiParams e, const float* __restrict__ part,
                                                    int splits) {
    const int groups = (e.N + 7) / 8;
    const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= static_cast<size_t>(groups) * e.M) return;
    const int m = static_cast<int>(i / groups), n = static_cast<int>(i - static_cast<size_t>(m) * groups) * 8;
    const EpiCols cols = epi_cols<F8>(e, n);
    const EpiToken t = epi_token<F8>(e, m, n);
    const size_t MN = static_cast<size_t>(e.M) * e.N;
    const float* at = part + static_cast<size_t>(m) * e.N + n;
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int k = 0; k < splits; ++k, at += MN) {
        if (n + 8 <= e.N) {
            const f32x4 a = *reinterpret_cast<const f32x4_rows*>(at);
            const f32x4 b = *reinterpret_cast<const f32x4_rows*>(at + 4);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[r] += a[r];
                s[4 + r] += b[r];
            }
        } else {
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (n + r < e.N) s[r] += at[r];
        }
    }
    epi_store<F8>(e, m, n, s, cols, t);
}

template <bool F8>
void launch_epi_wide(const EpiWideParams& p, int grid, int splits, bool once, hipStream_t s) {
    if (once)
        hipLaunchKernelGGL((gemm_epi_wide_kernel<F8, true>), dim3(grid, splits), dim3(512), 0, s, p);
    else
        hipLaunchKernelGGL((gemm_epi_wide_kernel<F8, false>), dim3(grid, splits), dim3(512), 0, s, p);
}

}  // namespace

namespace dev {

bool gemm_epi_sum(const EpiParams& e, const float* part, int splits, uint64_t stream,
                         std::string* err) {
    const size_t n = static_cast<size_t>((e.N + 7) / 8) * e.M;
    hipLaunchKernelGGL(e.xs != nullptr ? sum_partials_epi<true> : sum_partials_epi<false>,
                       dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0,
                       reinterpret_cast<hipStream_t>(stream), e, part, splits);
    KCMM_HIP_CHECK(hipGetLastError(), err);
    return true;
}

// The plan of the bf16 product of as many bytes: chunks cost the same here for
// either type.  Its K splits are of equal length; from 32 lines on it is asked
// for a multiple of 8, and the last split is shorter (542 x 3700 x 10928, 171
// lines: unsplit 174 us).
GemmWidePlan gemm_epi_wide_plan(const EpiParams& p, int max_splits, bool forced) {
    const uint32_t lines = (p.kb + 127) / 128, round = lines >= 32 ? (lines + 7) / 8 * 8 : lines;
    if (round >= 2) {
        const GemmWidePlan plan = gemm_wide_plan(static_cast<uint32_t>(p.M), static_cast<uint32_t>(p.N),
                                                 round * 64, false, max_splits, forced);
        if (plan.splits >= 1) return plan;
    }
    GemmWidePlan none;
    none.us = HUGE_VAL;
    return none;
}

bool gemm_epi_wide(const EpiParams& e, const GemmWidePlan& c, float* part, uint64_t stream,
                   std::string* err) {
    EpiWideParams p{};
    p.e = e;
    const int lines = static_cast<int>((e.kb + 127) / 128);
    p.lines = (lines + std::max(1, c.splits) - 1) / std::max(1, c.splits);
    const int splits = (lines + p.lines - 1) / p.lines;   // (none of them empty)
    p.part = splits > 1 ? part : nullptr;
    if (splits > 1 && part == nullptr) {
        *err = "epilogue product: K splits need their partials";
        return false;
    }
    const int tiles_n = (e.N + 255) / 256;
    const int fb[2] = {c.fb0, c.fb1};
    p.nw[1] = std::min(c.nw1, tiles_n);
    p.nw[0] = tiles_n - p.nw[1];
    int grid = 0;
    for (int z = 0; z < 2; ++z) {
        if (fb[z] < 1 || fb[z] > 4) {
            *err = "epilogue product: token tiles are 64, 128, 192 or 256 high";
            return false;
        }
        p.fb[z] = fb[z];
        p.full[z] = e.M / (64 * fb[z]);
        p.rag[z] = (e.M - p.full[z] * 64 * fb[z] + 63) / 64;
        grid += p.nw[z] * (p.full[z] + (p.rag[z] > 0));
    }
    const bool once = e.M <= 64 * c.fb0 && c.nw1 == 0;   // one token tile
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (e.xs != nullptr) launch_epi_wide<true>(p, grid, splits, once, s);
    else launch_epi_wide<false>(p, grid, splits, once, s);
    KCMM_HIP_CHECK(hipGetLastError(), err);
    return splits == 1 || gemm_epi_sum(e, p.part, splits, stream, err);
}

}  // namespace dev
}  // namespace kcmm
