// Rows as e4m3 codes with one fp32 scale per row, for products that read 8-bit
// activations (gemm_epi.hip).  Three sources of a row's values v (fp32, never
// rounded to bf16 on the way):
//  * norm:  h = bf16(x + residual), or x; v = h / sqrt(mean(h^2) + eps) * w;
//  * quant: v = x;
//  * silu:  v = silu(gate) * up of the fused [gate | up] row.
// Then a = max |v| over the finite v, scale = max(a / 448, 2^-126) (1 where a
// is 0), code = e4m3(v / scale): nearest even of the fp32 quotient, infinities
// at the largest code, NaN as NaN.  The scale keeps fp32, the codes are the
// one rounding to fewer bits, relative 2^-4, that the 8-bit product is for.
//
// Bound by memory for many rows (residual + norm of 8192 x 4096, 235 MB that no
// cache holds, 46.3 us = 5.1 TB/s; SwiGLU of 2048 x 14336 31.7 us = 4.6; a large copy
// moves 5.0) and by a launch and two dependent reductions for few (3.1 us in a
// graph for one row of 4096).  A row is read once: its values stay in registers between the sum, the
// maximum and the codes.
#include <algorithm>

#include "../device_api.hpp"
#include "common.hpp"
#include "fp8_page.hpp"

namespace kcmm {
namespace {

constexpr int kRowNorm = 0, kRowQuant = 1, kRowSilu = 2;

struct RowParams {
    const uint16_t* x;       // [rows][cols]; silu: [rows][2 cols], gate then up
    const uint16_t* r;       // norm: residual [rows][cols] or null
    const uint16_t* w;       // norm: [cols]
    uint16_t* hidden;        // norm with residual: [rows][cols]
    uint8_t* codes;          // [rows][cols]
    float* scales;           // [rows]
    int rows, cols;
    float eps;
};

__device__ __forceinline__ void widen8(const u32x4& v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(v[i] << 16);
        f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
}

// silu(g) u for g < -87: g e^g u (1 + e^g is 1 in fp32).  e^g goes below fp32 where a
// large u brings the product back, so e^g = 2^n 2^f, and 2^n comes last, on the product
// of the rest (2^-10 of it, which no u takes past fp32).  From g = -512 on nothing is
// left for any finite u; an infinite u gives infinity for every finite g.
__device__ __forceinline__ float silu_mul_far(float g, float u) {
    const float c = fmaxf(g, -512.0f), n = rintf(c * 1.44269502f);
    const float e = __builtin_amdgcn_exp2f(fmaf(c, 1.92596299e-8f, fmaf(c, 1.44269502f, -n)));
    return ldexpf(0x1p-10f * c * e * u, static_cast<int>(n) + 10);
}

// silu(g) u of 8 columns.  e^-g is 2^hi by the hardware's exp2, with what the
// rounding of hi leaves out as a factor; the quotient by its reciprocal, each with
// one step of its residual, so that both are rounded as if exact but for rare
// last places.  |hi| >= 126 (an e^-g or a reciprocal outside the normal numbers,
// which the instructions take for 0, infinities, NaN) takes the library's functions, or
// the form above.  (2048 x 14336: 37.7 us with those everywhere, 33.9 with
// the guards on every element; with the reciprocal alone three times the wrong
// codes.)
__device__ __forceinline__ void silu_mul8(float (&g)[8], const float (&u)[8]) {
    bool in = true;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float hi = g[e] * -1.44269502f;
        const float lo = fmaf(g[e], -1.92596299e-8f, fmaf(g[e], -1.44269502f, -hi));
        const float x = __builtin_amdgcn_exp2f(hi);
        const float s = 1.0f + fmaf(x, lo * 0.693147181f, x);
        const float r0 = __builtin_amdgcn_rcpf(s);
        const float r = fmaf(fmaf(-s, r0, 1.0f), r0, r0);
        const float q = g[e] * r;
        v[e] = fmaf(fmaf(-s, q, g[e]), r, q) * u[e];
        in &= fabsf(hi) < 126.0f;
    }
    if (__builtin_expect(!in, 0)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool far = g[e] < -87.0f && g[e] > -__builtin_inff();
            v[e] = far ? silu_mul_far(g[e], u[e]) : g[e] / (1.0f + expf(-g[e])) * u[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = v[e];
}

// The row's values before the norm's factor: piece `i` (8 columns) of row
// `row`.  norm: stores the hidden piece where there is a residual.
template <int MODE>
__device__ __forceinline__ void row_piece(const RowParams& p, size_t row, int i, float (&v)[8]) {
    if constexpr (MODE == kRowSilu) {
        const uint16_t* g = p.x + row * 2 * p.cols + i * 8;
        float u[8];
        widen8(*reinterpret_cast<const u32x4*>(g), v);
        widen8(*reinterpret_cast<const u32x4*>(g + p.cols), u);
        silu_mul8(v, u);
    } else {
        const size_t at = row * p.cols + i * 8;
        widen8(*reinterpret_cast<const u32x4*>(p.x + at), v);
        if constexpr (MODE == kRowNorm) {
            if (p.r == nullptr) return;
            float r[8];
            widen8(*reinterpret_cast<const u32x4*>(p.r + at), r);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
            const u32x4 h = pack_bf16x8(v);
            *reinterpret_cast<u32x4*>(p.hidden + at) = h;
            widen8(h, v);   // the norm is that of the stored row
        }
    }
}

// The largest |v| (of those that are no NaN: the hardware's maximum passes it
// over), and that of the finite ones.
__device__ __forceinline__ float amax8(const float (&v)[8], float a) {
#pragma unroll
    for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(v[e]));
    return a;
}
__device__ __forceinline__ float finite_amax8(const float (&v)[8], float a) {
#pragma unroll
    for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(v[e]) < __builtin_inff() ? fabsf(v[e]) : 0.0f);
    return a;
}

__device__ __forceinline__ float row_scale(float a) {
    return a > 0.0f ? fmaxf(a / 448.0f, 0x1p-126f) : 1.0f;
}

// Eight values as codes; r = 1 / scale; finite: the row has no infinity.
__device__ __forceinline__ u32x2 row_codes(const float (&v)[8], float scale, float r, bool finite) {
    u32x2 o;
    bool plain = finite && scale >= kFp8QuotientMin && scale <= kFp8QuotientMax;
#pragma unroll
    for (int e = 0; e < 4; ++e) plain &= !__builtin_isunordered(v[2 * e], v[2 * e + 1]);
    if (__builtin_expect(plain, 1)) {
        float q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = fp8_quotient(v[e], scale, r);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * w], q[4 * w + 1], 0, false);
            o[w] = static_cast<uint32_t>(
                __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * w + 2], q[4 * w + 3], lo, true));
        }
        return o;
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        o[w] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[w] |= f32_to_fp8e4m3(v[4 * w + e] / scale) << (8 * e);
    }
    return o;
}

// Sum (or maximum) over a row's WPR waves, waves in order; `red` holds WPR
// floats of this row.  A second use needs other floats.
template <int WPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red, int wave) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float u = __shfl_xor(v, o);
        v = MAX ? fmaxf(v, u) : v + u;
    }
    if constexpr (WPR == 1) return v;
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int w = 1; w < WPR; ++w) s = MAX ? fmaxf(s, red[w]) : s + red[w];
    return s;
}

// A row whose squares leave fp32 (a sum past 2^128, or one with eps under
// 2^-100, where squares lose bits) is normed as 2^-80 or 2^80 times itself,
// with eps times the square of that: the same v.  1 for any other row.
__device__ __forceinline__ float norm_rescale(float ss, float eps) {
    if (!(ss < __builtin_inff())) return 0x1p-80f;
    return ss + eps < 0x1p-100f ? 0x1p80f : 1.0f;
}

template <int P>
__device__ __forceinline__ float squares(const float (&v)[P][8]) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += v[i][e] * v[i][e];
    return ss;
}

// WPR waves a row, RPW rows a workgroup, at most P pieces of 8 columns a
// lane (cols <= 512 * WPR * P).
template <int MODE, int WPR, int P, int RPW>
__global__ __launch_bounds__(64 * WPR * RPW) void quant_rows(RowParams p) {
    static_assert(WPR == 1 || RPW == 1, "a barrier is all of one row's");
    __shared__ float red[4][RPW][WPR];
    const int slot = threadIdx.x / (64 * WPR), t = threadIdx.x % (64 * WPR), wave = t >> 6;
    const bool live = blockIdx.x * RPW + slot < static_cast<unsigned>(p.rows);
    const size_t row = live ? blockIdx.x * RPW + slot : 0;
    const int n = live ? p.cols / 8 : 0;
    float v[P][8];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int at = t + i * 64 * WPR;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
        if (at < n) row_piece<MODE>(p, row, at, v[i]);
    }
    if constexpr (MODE == kRowNorm) {
        float w[P][8], eps = p.eps;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int at = t + i * 64 * WPR;
            widen8(*reinterpret_cast<const u32x4*>(p.w + (at < n ? at : 0) * 8), w[i]);
        }
        float ss = row_reduce<WPR, false>(squares(v), red[0][slot], wave);
        const float up = norm_rescale(ss, eps);
        if (__builtin_expect(up != 1.0f, 0)) {   // the same for all of the row's threads
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] *= up;
            ss = row_reduce<WPR, false>(squares(v), red[2][slot], wave);
            eps = eps * up * up;
        }
        const float f = 1.0f / sqrtf(ss / static_cast<float>(p.cols) + eps);
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * f * w[i][e];
    }
    float a = 0.0f;   // (a piece past the row's end is zeros)
#pragma unroll
    for (int i = 0; i < P; ++i) a = amax8(v[i], a);
    a = row_reduce<WPR, true>(a, red[1][slot], wave);
    const bool finite = a < __builtin_inff();
    if (__builtin_expect(!finite, 0)) {   // the same for all of the row's threads
        a = 0.0f;
#pragma unroll
        for (int i = 0; i < P; ++i) a = finite_amax8(v[i], a);
        a = row_reduce<WPR, true>(a, red[3][slot], wave);
    }
    const float scale = row_scale(a), r = 1.0f / scale;
    if (live && t == 0) p.scales[row] = scale;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int at = t + i * 64 * WPR;
        if (at < n)
            *reinterpret_cast<u32x2*>(p.codes + row * p.cols + at * 8) = row_codes(v[i], scale, r, finite);
    }
}

// Rows too long for the registers of 16 waves: each pass reads the row again
// (from L2), the norm's from the hidden row where there is one.
template <int MODE>
__global__ __launch_bounds__(1024) void quant_long_rows(RowParams p) {
    __shared__ float red[4][16];
    const size_t row = blockIdx.x;
    const int n = p.cols / 8, t = threadIdx.x, wave = t >> 6;
    float f = 1.0f, up = 1.0f, a = 0.0f, v[8], w[8];
    RowParams q = p;
    if constexpr (MODE == kRowNorm) {
        auto squares = [&](float* at) {
            float ss = 0.0f;
            for (int i = t; i < n; i += 1024) {
                row_piece<MODE>(q, row, i, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += v[e] * up * (v[e] * up);
            }
            if (p.r != nullptr) {   // from now on a thread reads what it wrote itself
                q.x = p.hidden;
                q.r = nullptr;
            }
            return row_reduce<16, false>(ss, at, wave);
        };
        float ss = squares(red[0]);
        up = norm_rescale(ss, p.eps);
        if (up != 1.0f) ss = squares(red[2]);
        f = 1.0f / sqrtf(ss / static_cast<float>(p.cols) + p.eps * up * up);
    }
    auto value = [&](int i) {
        row_piece<MODE>(q, row, i, v);
        if constexpr (MODE == kRowNorm) {
            widen8(*reinterpret_cast<const u32x4*>(p.w + i * 8), w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] * up * f * w[e];
        }
    };
    for (int i = t; i < n; i += 1024) {
        value(i);
        a = amax8(v, a);
    }
    a = row_reduce<16, true>(a, red[1], wave);
    const bool finite = a < __builtin_inff();
    if (!finite) {
        a = 0.0f;
        for (int i = t; i < n; i += 1024) {
            value(i);
            a = finite_amax8(v, a);
        }
        a = row_reduce<16, true>(a, red[3], wave);
    }
    const float scale = row_scale(a), r = 1.0f / scale;
    if (t == 0) p.scales[row] = scale;
    for (int i = t; i < n; i += 1024) {
        value(i);
        *reinterpret_cast<u32x2*>(p.codes + row * p.cols + i * 8) = row_codes(v, scale, r, finite);
    }
}

template <int MODE, int WPR, int P>
void launch_rows(const RowParams& p, hipStream_t s) {
    constexpr int RPW = WPR == 1 ? 4 : 1;
    hipLaunchKernelGGL((quant_rows<MODE, WPR, P, RPW>), dim3((p.rows + RPW - 1) / RPW),
                       dim3(64 * WPR * RPW), 0, s, p);
}

// Up to 512 rows a piece a lane, for the shorter chain (512 x 4096 norm 5.7 us;
// two pieces a lane 6.0); more rows fill the chip, and half as many waves a row
// wait less at its reductions (one piece / two: norm of 8192 x 4096 42.7 / 42.5 us,
// 8192 x 2816 38.2 / 33.3, 8192 x 1024 15.0 / 14.6, quant of 8192 x 4096 22.0 / 18.9).
template <int MODE>
bool quant(const RowParams& p, uint64_t stream, std::string* err) {
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int n = p.cols / 8;   // pieces of a row
    const bool few = p.rows <= 512;
    if (n <= 64) launch_rows<MODE, 1, 1>(p, s);
    else if (few && n <= 128) launch_rows<MODE, 2, 1>(p, s);
    else if (few && n <= 256) launch_rows<MODE, 4, 1>(p, s);
    else if (few && n <= 512) launch_rows<MODE, 8, 1>(p, s);
    else if (few && n <= 1024) launch_rows<MODE, 16, 1>(p, s);
    else if (n <= 128) launch_rows<MODE, 1, 2>(p, s);
    else if (n <= 256) launch_rows<MODE, 2, 2>(p, s);
    else if (n <= 512) launch_rows<MODE, 4, 2>(p, s);
    else if (n <= 1024) launch_rows<MODE, 8, 2>(p, s);
    else if (n <= 2048) launch_rows<MODE, 16, 2>(p, s);
    else if (n <= 4096) launch_rows<MODE, 16, 4>(p, s);
    else hipLaunchKernelGGL(quant_long_rows<MODE>, dim3(p.rows), dim3(1024), 0, s, p);
    KCMM_HIP_CHECK(hipGetLastError(), err);
    return true;
}

RowParams row_params(uint64_t x, uint64_t codes, uint64_t scales, uint32_t rows, uint32_t cols) {
    RowParams p{};
    p.x = reinterpret_cast<const uint16_t*>(x);
    p.codes = reinterpret_cast<uint8_t*>(codes);
    p.scales = reinterpret_cast<float*>(scales);
    p.rows = static_cast<int>(rows);
    p.cols = static_cast<int>(cols);
    return p;
}

}  // namespace

namespace dev {

bool add_rmsnorm_fp8(uint64_t x, uint64_t residual, uint64_t w, uint64_t hidden, uint64_t codes,
                     uint64_t scales, uint32_t rows, uint32_t cols, float eps, uint64_t stream,
                     std::string* err) {
    RowParams p = row_params(x, codes, scales, rows, cols);
    p.r = reinterpret_cast<const uint16_t*>(residual);
    p.w = reinterpret_cast<const uint16_t*>(w);
    p.hidden = reinterpret_cast<uint16_t*>(hidden);
    p.eps = eps;
    return quant<kRowNorm>(p, stream, err);
}

bool quant_rows_fp8(uint64_t x, uint64_t codes, uint64_t scales, uint32_t rows, uint32_t cols,
                    uint64_t stream, std::string* err) {
    return quant<kRowQuant>(row_params(x, codes, scales, rows, cols), stream, err);
}

bool silu_mul_fp8(uint64_t gate_up, uint64_t codes, uint64_t scales, uint32_t rows, uint32_t inter,
                  uint64_t stream, std::string* err) {
    return quant<kRowSilu>(row_params(gate_up, codes, scales, rows, inter), stream, err);
}

}  // namespace dev
}  // namespace kcmm
