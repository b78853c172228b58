// Low-rank adapters of many requests beside a shared projection (gfx950):
//   y[t] = bf16(base[t] + (scale_a x[t] A_a^T) B_a^T),  a = adapter_ids[t],
// A_a [slices * rank][k] and B_a [n][rank] bf16; column n takes the rank values
// of its slice.  A token without an adapter keeps base.  Two kernels: the low-rank
// values v = scale x A^T go through memory of the caller's; y is rounded once.
//
// The first works on 16 tokens a block, in the order in which they come, and so does
// the second for few tokens and for large prompts: a block's tokens may have any
// adapters, and each of these takes its turn with all 16 columns of the matrix
// instruction, of which only its own tokens' are kept (a column's values come from its own
// token alone, so what another token or adapter holds, infinities too, goes nowhere).
// Prompts have one adapter a block, decode batches up to 16, whose weights are then what
// has to be read, once a block.  Hundreds of tokens go through the second product by
// units: up to 16 tokens of one adapter out of 64.
//  * shrink: k dealt to the waves of a workgroup by lines of 128 bytes, their sums
//    joined in LDS, in wave order.  A workgroup has 16 or 32 rows of A and one of the
//    block's adapters, or several in turn.  Bound by what one CU loads (64 bytes a
//    cycle).
//  * expand: bound by base and y in HBM for prompts, by latency for few tokens.  The
//    matrix instruction has 32 consecutive k and a rank seldom fills them, so the
//    second parts of the values (below) are nearly free.
// A CU's load path takes 8 lanes with one line of 128 bytes in 2 cycles but 8 lanes with a
// line each in 8: operands read from rows straight into the matrix instruction's
// layout cost 4 times the cycles of whole lines.  Hence the way through LDS in the
// shrink, the layout of the low-rank values, and tokens as rows in the expand (3001
// tokens, rank 32, k 4096, n 28672: 36 + 116 us with such reads, 11 + 70 without; the
// 70 are 4.9 TB/s of base and y).
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "../device_api.hpp"
#include "common.hpp"

namespace kcmm {
namespace {

struct LoraParams {
    const uint16_t* x;
    const uint16_t* a;
    const uint16_t* b;
    const float* scales;
    const int32_t* ids;
    float* low;
    const uint16_t* base;
    uint16_t* y;
    int m, n, k, adapters, rank, slices, rows;   // rows = slices * rank
    int ends[4];                                 // of the slices' columns
    int chunks[4];                               // end of the slices' column chunks
};

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                   0, 0, 0);
}

// Adapter of token t, or -1.
__device__ __forceinline__ int adapter_of(const LoraParams& p, int t) {
    const int id = t < p.m ? p.ids[t] : -1;
    return static_cast<uint32_t>(id) < static_cast<uint32_t>(p.adapters) ? id : -1;
}

// Takes the first adapter of the tokens still to be served out of their set: a bit
// for each of the block's tokens; -1 when none is left.
__device__ __forceinline__ int next_adapter(int id, uint32_t* left) {
    if (*left == 0) return -1;
    const int a = __builtin_amdgcn_readlane(id, __ffs(static_cast<int>(*left)) - 1);
    *left &= ~static_cast<uint32_t>(__ballot(id == a));
    return a;
}

// The units of a block of 64 tokens: up to 16 tokens of one adapter, in the order of
// their adapters' first tokens; a lane a token.
struct Units {
    int id;          // this lane's token's adapter
    uint64_t left;   // tokens whose adapter's turn has not come
    uint64_t ours = 0;   // those of the adapter that has it
    int a = -1, from = 0, count = 0;
    __device__ Units(const LoraParams& p, int t0, int lane) : id(adapter_of(p, t0 + lane)) {
        left = __ballot(id >= 0);
    }
    // false: no more of them
    __device__ bool next() {
        from += 16;
        if (from >= __popcll(ours)) {
            if (left == 0) return false;
            a = __builtin_amdgcn_readlane(id, __ffsll(static_cast<long long>(left)) - 1);
            ours = __ballot(id == a);
            left &= ~ours;
            from = 0;
        }
        count = min(16, __popcll(ours) - from);
        return true;
    }
    // token (0 .. 63) of column l & 15; a column behind the last has the first one's
    __device__ int column(int lane) const {
        const int nth = __popcll(ours & ((1ull << lane) - 1)) - from;
        const bool mine = id == a && nth >= 0 && nth < 16;
        const int at = __builtin_amdgcn_ds_permute(4 * (mine ? nth : 63), lane);
        return __shfl(at, (lane & 15) < count ? lane & 15 : 0);
    }
};

// Rows of 128 bytes of k in LDS, one wave's own: piece j of 16 bytes of row r lies at
// r * 128 + 16 (j ^ (r & 7)), so that writes of whole rows and reads of one piece of
// 16 rows both pass all banks.
__device__ __forceinline__ u32x4* piece_at(u32x4* rows, int row, int piece) {
    return rows + row * 8 + (piece ^ (row & 7));
}

// Low-rank values, 4 bytes each, of a block of 16 tokens (`count` of them in the last
// block), in the order in which the second product reads them: by slices, 2 P pieces
// of 8 values (P = rank / 8) of all tokens side by side; the first P their bf16
// values, the others what these leave, bf16 too.  2^-16 of a value is lost so, a 2^-8th
// of what the rounding of y is.
struct LowBlock {
    u32x4* at;
    int count;
    __device__ LowBlock(const LoraParams& p, int block, int slice)
        : at(reinterpret_cast<u32x4*>(p.low + static_cast<size_t>(block) * 16 * p.rows)),
          count(min(16, p.m - 16 * block)) {
        at += slice * (p.rank / 4) * count;
    }
    __device__ u32x4* piece(int q, int token) const { return at + q * count + token; }
};

// Workgroup (block of 16 tokens, turn, row group): R low-rank rows for the turn-th,
// turn + turns-th ... of the block's adapters.  The adapter's tokens are the first
// columns, so that up to 8 of them take one load a line.  A wave loads lines of
// 128 bytes, 8 lanes a row, U of them before it uses the first.
template <int R, int U>
__global__ __launch_bounds__(512) void lora_shrink(LoraParams p, int turns) {
    constexpr int NW = 8, RB = R / 16, WL = R / 8;   // waves; products, loads of weights a line
    __shared__ u32x4 s_rows[NW][(2 + WL) * 64];
    const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    u32x4* const rows = s_rows[wave];
    const int t0 = blockIdx.x * 16, row0 = blockIdx.z * R;
    const int id = adapter_of(p, t0 + ln);
    uint32_t left = static_cast<uint32_t>(__ballot(id >= 0)) & 0xffffu;
    const int pieces = p.k / 8, lines = (pieces + 7) / 8;
    for (int turn = 0;; ++turn) {
        const int a = next_adapter(id, &left);
        if (a < 0) break;
        if (turn % turns != static_cast<int>(blockIdx.y)) continue;
        // token of the block that column `lane` has; a column behind the last takes the
        // first one's along
        const uint32_t ours = static_cast<uint32_t>(__ballot(id == a)) & 0xffffu;
        const int count = __popc(ours), nth = __popc(ours & ((1u << ln) - 1));
        const int token = __builtin_amdgcn_ds_permute(4 * (lane < 16 && id == a ? nth : 63), ln);
        const uint16_t* xs[2];
        const uint16_t* ws[WL];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = 8 * i + (lane >> 3);
            xs[i] = p.x + static_cast<size_t>(t0 + __shfl(token, c < count ? c : 0)) * p.k;
        }
#pragma unroll
        for (int i = 0; i < WL; ++i)
            ws[i] = p.a + (static_cast<size_t>(a) * p.rows + min(row0 + 8 * i + (lane >> 3), p.rows - 1)) * p.k;
        f32x4 sum[RB];
#pragma unroll
        for (int i = 0; i < RB; ++i) sum[i] = f32x4{0, 0, 0, 0};
        // Lines l, l + NW ... l + (U - 1) NW; the last ones may be partial or past the row
        auto lines_of = [&](int l, auto XL, auto tail) __attribute__((always_inline)) {
            u32x4 x[U][XL], w[U][WL];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int piece = (l + u * NW) * 8 + (lane & 7);
                const uint32_t at = static_cast<uint32_t>(tail && piece >= pieces ? 0 : piece) * 8;
#pragma unroll
                for (int i = 0; i < XL; ++i) x[u][i] = *reinterpret_cast<const u32x4*>(xs[i] + at);
#pragma unroll
                for (int i = 0; i < WL; ++i) w[u][i] = *reinterpret_cast<const u32x4*>(ws[i] + at);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = !tail || (l + u * NW) * 8 + (lane & 7) < pieces;
                const u32x4 none = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < XL; ++i) *piece_at(rows, 8 * i + (lane >> 3), lane & 7) = in ? x[u][i] : none;
#pragma unroll
                for (int i = 0; i < WL; ++i)
                    *piece_at(rows, 8 * (XL + i) + (lane >> 3), lane & 7) = in ? w[u][i] : none;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // (with 8 columns loaded the others are these again)
                    const u32x4 xf = *piece_at(rows, XL == 1 ? ln & 7 : ln, 4 * h + lg);
#pragma unroll
                    for (int i = 0; i < RB; ++i)
                        sum[i] = mfma(*piece_at(rows, 8 * XL + 16 * i + ln, 4 * h + lg), xf, sum[i]);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        };
        auto all_lines = [&](auto XL) __attribute__((always_inline)) {
            int l = wave;
#pragma clang loop unroll(disable)
            for (; (l + (U - 1) * NW + 1) * 8 <= pieces; l += NW * U) lines_of(l, XL, std::false_type{});
            if (l < lines) lines_of(l, XL, std::true_type{});
        };
        if (count <= 8) all_lines(std::integral_constant<int, 1>{});
        else all_lines(std::integral_constant<int, 2>{});
        // the waves' sums, each in the place of its lines
#pragma unroll
        for (int i = 0; i < RB; ++i) rows[i * 64 + lane] = __builtin_bit_cast(u32x4, sum[i]);
        __syncthreads();
        const float scale = p.scales != nullptr ? p.scales[a] : 1.0f;
        const int t = __shfl(token, ln);
        for (int i = wave; i < RB; i += NW) {
            f32x4 v = {0, 0, 0, 0};
            for (int j = 0; j < NW; ++j) v += __builtin_bit_cast(f32x4, s_rows[j][i * 64 + lane]);
            float part[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (the last fp32 values would round to an infinity: the largest bf16 instead, so
                // that they too leave what the second part holds; an infinity leaves nothing)
                constexpr float kMost = 3.38953139e38f;
                v[e] *= scale;
                part[e] = fabsf(v[e]) < INFINITY ? bf16_round_hw(fminf(fmaxf(v[e], -kMost), kMost)) : v[e];
                part[4 + e] = fabsf(part[e]) < INFINITY ? v[e] - part[e] : 0.0f;
            }
            // rows 4 lg .. +3 of each 16, of column ln: half a piece
            const int row = row0 + 16 * i + 4 * lg;
            if (ln < count && row < p.rows) {
                const int slice = row / p.rank, q = (row - slice * p.rank) / 8;
                const LowBlock low(p, blockIdx.x, slice);
                const u32x4 o = pack_bf16x8(part);
                reinterpret_cast<u32x2*>(low.piece(q, t))[row >> 2 & 1] = u32x2{o[0], o[1]};
                reinterpret_cast<u32x2*>(low.piece(p.rank / 8 + q, t))[row >> 2 & 1] = u32x2{o[2], o[3]};
            }
        }
        __syncthreads();
    }
}

// The columns of a chunk: `width` of one slice.
struct Columns {
    int slice, n0, end;
    __device__ bool find(const LoraParams& p, int chunk, int width) {
        slice = 0;
        while (slice < p.slices && chunk >= p.chunks[slice]) ++slice;
        if (slice == p.slices) return false;
        end = p.ends[slice];
        n0 = (slice > 0 ? p.ends[slice - 1] : 0) + (chunk - (slice > 0 ? p.chunks[slice - 1] : 0)) * width;
        return true;
    }
};

// The piece of a token's values that lane group lg has in step k, and the piece of the
// weights that goes with it.
struct Piece {
    int value, weight;
    bool in;
    __device__ Piece(int k, int lg, int P) {
        in = 4 * k + lg < 2 * P;
        value = in ? 4 * k + lg : 0;
        weight = value < P ? value : value - P;
    }
};

__device__ __forceinline__ float bf16_half(uint32_t pair, int which) {
    return __uint_as_float(which ? pair & 0xffff0000u : pair << 16);
}

// Few tokens: a wave has 16 of them and 16 columns, and the weights of U adapters on
// their way at once.
template <int STEPS>
__global__ __launch_bounds__(256) void lora_expand_few(LoraParams p) {
    constexpr int U = STEPS <= 2 ? 8 : 4;
    const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    Columns columns;
    if (!columns.find(p, blockIdx.x * 4 + wave, 16)) return;
    const int t = blockIdx.y * 16 + ln, P = p.rank / 8;
    const int id = adapter_of(p, t);
    uint32_t left = static_cast<uint32_t>(__ballot(id >= 0)) & 0xffffu;
    const size_t at = static_cast<size_t>(min(t, p.m - 1)) * p.n + columns.n0 + 4 * lg;
    const u32x2 base = *reinterpret_cast<const u32x2*>(p.base + at);
    const LowBlock low(p, blockIdx.y, columns.slice);
    const uint16_t* const w = p.b + static_cast<size_t>(columns.n0 + ln) * p.rank;
    u32x4 vf[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        const Piece q(k, lg, P);
        vf[k] = *low.piece(q.value, min(ln, low.count - 1));
        if (!q.in) vf[k] = u32x4{0, 0, 0, 0};
    }
    f32x4 acc = {0, 0, 0, 0};
    while (left != 0) {
        int a[U];
        u32x4 wf[U][STEPS];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            a[u] = next_adapter(id, &left);
            if (a[u] < 0) continue;
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
                wf[u][k] = *reinterpret_cast<const u32x4*>(w + static_cast<size_t>(a[u]) * p.n * p.rank +
                                                          Piece(k, lg, P).weight * 8);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (a[u] < 0) continue;
            f32x4 d = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
                d = mfma(Piece(k, lg, P).in ? wf[u][k] : u32x4{0, 0, 0, 0}, vf[k], d);
            if (id == a[u]) acc = d;
        }
    }
    if (t >= p.m) return;
    u32x2 out = base;
    if (id >= 0) {
        float v[8] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = bf16_half(base[e >> 1], e & 1) + acc[e];
        const u32x4 o = pack_bf16x8(v);
        out = u32x2{o[0], o[1]};
    }
    *reinterpret_cast<u32x2*>(p.y + at) = out;
}

// Hundreds of tokens: a wave has 16 columns and the units of 64 tokens, one after the
// other, each with a load of its adapter's weights: mixed adapters load them for 16 of their
// tokens at a time, not for each block of 16 tokens that holds one.
template <int STEPS>
__global__ __launch_bounds__(256) void lora_expand_units(LoraParams p) {
    const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    Columns columns;
    if (!columns.find(p, blockIdx.x * 4 + wave, 16)) return;
    const int t0 = blockIdx.y * 64, P = p.rank / 8, column = columns.n0 + 4 * lg;
    Units unit(p, t0, lane);
    // tokens without an adapter keep base
    if (p.y != p.base) {
        uint64_t none = ~unit.left;
        if (p.m - t0 < 64) none &= (1ull << (p.m - t0)) - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const size_t at = static_cast<size_t>(t0 + 16 * i + ln) * p.n + column;
            if (none >> (16 * i + ln) & 1)
                *reinterpret_cast<u32x2*>(p.y + at) = *reinterpret_cast<const u32x2*>(p.base + at);
        }
    }
    while (unit.next()) {
        const int token = unit.column(lane);
        const size_t at = static_cast<size_t>(t0 + token) * p.n + column;
        const u32x2 base = *reinterpret_cast<const u32x2*>(p.base + at);
        const LowBlock low(p, 4 * blockIdx.y + (token >> 4), columns.slice);
        const uint16_t* const w =
            p.b + (static_cast<size_t>(unit.a) * p.n + columns.n0 + ln) * p.rank;
        u32x4 vf[STEPS], wf[STEPS];
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            const Piece q(k, lg, P);
            vf[k] = *low.piece(q.value, token & 15);
            wf[k] = *reinterpret_cast<const u32x4*>(w + q.weight * 8);
        }
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            const u32x4 none = {0, 0, 0, 0};
            const bool in = Piece(k, lg, P).in;
            acc = mfma(in ? wf[k] : none, in ? vf[k] : none, acc);
        }
        float v[8] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = bf16_half(base[e >> 1], e & 1) + acc[e];
        const u32x4 o = pack_bf16x8(v);
        if (ln < unit.count) *reinterpret_cast<u32x2*>(p.y + at) = u32x2{o[0], o[1]};
    }
}

// Many tokens: a wave has NB * 16 columns and runs through `per` blocks of 16 tokens.
// The tokens are the rows of its products, lane ln has the NB columns from ln * NB on, so
// that 16 lanes read and write whole lines of base and y; the weights stay in registers
// for as long as the adapter does, the next block's base and values are on their way
// while one is worked on.
template <int NB, int STEPS>
__global__ __launch_bounds__(256) void lora_expand(LoraParams p, int per) {
    typedef uint32_t Run __attribute__((ext_vector_type(NB / 2)));   // NB columns
    const int lane = threadIdx.x & 63, ln = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    Columns columns;
    if (!columns.find(p, blockIdx.x * 4 + wave, NB * 16)) return;
    const int P = p.rank / 8, blocks = (p.m + 15) / 16;
    const int first = blockIdx.y * per, behind = min(first + per, blocks);
    // past the slice's end its last columns, which are not stored
    const bool stored = columns.n0 + ln * NB < columns.end;
    const int column = min(columns.n0 + ln * NB, columns.end - NB);
    const uint16_t* const w = p.b + static_cast<size_t>(column) * p.rank;

    struct Block {
        int id;
        Run base[4];   // of tokens 4 lg .. +3
        u32x4 v[STEPS];
    };
    auto load = [&](int block) __attribute__((always_inline)) {
        Block r;
        r.id = adapter_of(p, block * 16 + ln);
        const LowBlock low(p, block, columns.slice);
#pragma unroll
        for (int k = 0; k < STEPS; ++k) r.v[k] = *low.piece(Piece(k, lg, P).value, min(ln, low.count - 1));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r.base[i] = __builtin_nontemporal_load(reinterpret_cast<const Run*>(
                p.base + static_cast<size_t>(min(block * 16 + 4 * lg + i, p.m - 1)) * p.n + column));
        return r;
    };
    int held = -1;
    u32x4 wf[NB][STEPS];
    auto finish = [&](int block, const Block& r) __attribute__((always_inline)) {
        f32x4 acc[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = f32x4{0, 0, 0, 0};
        const uint32_t any = static_cast<uint32_t>(__ballot(r.id >= 0)) & 0xffffu;
        uint32_t left = any;
        for (int a = next_adapter(r.id, &left); a >= 0; a = next_adapter(r.id, &left)) {
            if (a != held) {
                held = a;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int k = 0; k < STEPS; ++k) {
                        wf[b][k] = *reinterpret_cast<const u32x4*>(
                            w + (static_cast<size_t>(a) * p.n + b) * p.rank + Piece(k, lg, P).weight * 8);
                        if (!Piece(k, lg, P).in) wf[b][k] = u32x4{0, 0, 0, 0};
                    }
                // (here, and not for all loads after each block)
                __builtin_amdgcn_s_waitcnt(0x0f70);
            }
            const uint32_t ours = static_cast<uint32_t>(__ballot(r.id == a)) >> (4 * lg);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                f32x4 d = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < STEPS; ++k)
                    d = mfma(Piece(k, lg, P).in ? r.v[k] : u32x4{0, 0, 0, 0}, wf[b][k], d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (ours >> i & 1) acc[b][i] = d[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = block * 16 + 4 * lg + i;
            float v[8] = {};
#pragma unroll
            for (int b = 0; b < NB; ++b) v[b] = bf16_half(r.base[i][b >> 1], b & 1) + acc[b][i];
            const u32x4 o = pack_bf16x8(v);
            Run out;
#pragma unroll
            for (int e = 0; e < NB / 2; ++e) out[e] = any >> (4 * lg + i) & 1 ? o[e] : r.base[i][e];
            if (t < p.m && stored)
                __builtin_nontemporal_store(out, reinterpret_cast<Run*>(p.y + static_cast<size_t>(t) * p.n + column));
        }
    };
    Block one = load(first);
    for (int block = first; block < behind; block += 2) {
        const Block two = load(min(block + 1, behind - 1));
        finish(block, one);
        one = load(min(block + 2, behind - 1));
        if (block + 1 < behind) finish(block + 1, two);
    }
}

template <int R, int U>
void launch_shrink(const LoraParams& p, hipStream_t s) {
    const int blocks = (p.m + 15) / 16, groups = (p.rows + R - 1) / R;
    const int turns = std::max(1, std::min({16, p.m, p.adapters, 512 / (blocks * groups)}));
    hipLaunchKernelGGL((lora_shrink<R, U>), dim3(blocks, turns, groups), dim3(512), 0, s, p, turns);
}

// Chunks of `width` columns; returns their number.
int deal_columns(LoraParams& p, int width) {
    int chunks = 0;
    for (int i = 0; i < p.slices; ++i) {
        chunks += (p.ends[i] - (i > 0 ? p.ends[i - 1] : 0) + width - 1) / width;
        p.chunks[i] = chunks;
    }
    return chunks;
}

template <int NB, int STEPS>
void launch_expand(LoraParams& p, hipStream_t s) {
    const int chunks = deal_columns(p, 16 * NB);
    const long long blocks = (p.m + 15) / 16;
    const int per = static_cast<int>(std::max<long long>(1, std::min<long long>(16, blocks * chunks / 4096)));
    const dim3 grid((chunks + 3) / 4, static_cast<unsigned>((blocks + per - 1) / per));
    hipLaunchKernelGGL((lora_expand<NB, STEPS>), grid, dim3(256), 0, s, p, per);
}

template <int NB, int STEPS>
void launch_expand_any(LoraParams& p, hipStream_t s) {
    // Runs of blocks pay once base and y are large.  Units and this, the whole call, k 4096,
    // tokens in runs of 8 adapters, ranks 16 / 64: 1024 tokens, n 6144 21.5 and 21.6 us /
    // 40.4 and 41.6; from 2048 tokens, n 4096 20.5 and 19.8 / 42.3 and 33.2 on, to 4096
    // tokens, n 28672 240 and 102 / 430 and 145.  (Where adapters are mixed, weights are
    // loaded anew for each block: 2048 tokens, n 4096 32.4 and 48.9 / 82.9 and 149.  Ids
    // lie on the device, so no rule can tell.)
    const long long blocks = (p.m + 15) / 16;
    if (blocks * ((p.n + 63) / 64) >= 8192) return launch_expand<NB, STEPS>(p, s);
    const int chunks = deal_columns(p, 16);
    // Units where there are waves enough without the latencies that the other form hides.
    // Few and units, as above, mixed: 512 tokens, n 4096 13.3 and 14.0 us / 45.2 and 28.5,
    // 1024 20.5 and 19.0 / 81.1 and 48.4; in runs of an adapter 10.0 and 10.7 / 16.9 and 17.0,
    // 14.9 and 14.1 / 26.1 and 25.8.  With fewer waves, 256 tokens, n 4096: mixed 10.8 and 12.6
    // / 26.8 and 19.4, runs 8.9 and 10.3 / 12.5 and 13.7; 64 tokens of 16 adapters, n 6144 12
    // and 17.
    const long long tiles = (p.m + 63) / 64;
    if (chunks * tiles >= 2048) {
        hipLaunchKernelGGL((lora_expand_units<STEPS>), dim3((chunks + 3) / 4, static_cast<unsigned>(tiles)), dim3(256), 0,
                           s, p);
        return;
    }
    hipLaunchKernelGGL((lora_expand_few<STEPS>), dim3((chunks + 3) / 4, static_cast<unsigned>(blocks)), dim3(256), 0, s,
                       p);
}

}  // namespace

namespace dev {

bool lora_add_bf16(const LoraArgs& a, std::string* err) {
    LoraParams p{};
    p.x = reinterpret_cast<const uint16_t*>(a.x);
    p.a = reinterpret_cast<const uint16_t*>(a.a);
    p.b = reinterpret_cast<const uint16_t*>(a.b);
    p.scales = reinterpret_cast<const float*>(a.scales);
    p.ids = reinterpret_cast<const int32_t*>(a.ids);
    p.low = reinterpret_cast<float*>(a.low);
    p.base = reinterpret_cast<const uint16_t*>(a.base);
    p.y = reinterpret_cast<uint16_t*>(a.y);
    p.m = static_cast<int>(a.m);
    p.n = static_cast<int>(a.n);
    p.k = static_cast<int>(a.k);
    p.adapters = static_cast<int>(a.adapters);
    p.rank = static_cast<int>(a.rank);
    p.slices = static_cast<int>(a.slices);
    p.rows = p.rank * p.slices;
    for (int i = 0; i < p.slices; ++i) p.ends[i] = static_cast<int>(a.slice_ends[i]);
    hipStream_t s = reinterpret_cast<hipStream_t>(a.stream);
    // Twice the rows a workgroup halve what the tokens cost it, but leave half as many
    // workgroups.  16 and 32 rows, the whole call: 64 tokens of 16 adapters, 48 rows,
    // k 4096: 11.7 and 12.9 us; 64 of 8, 64 rows, k 14336: 16.7 and 21.2; 512 (384
    // products): 22.8 and 24.2; 3001 prompt tokens (752): 85.2 and 83.3; 2048 tokens, 192
    // rows (1536): 69.1 and 62.7.  8 or 64 rows, or 16 waves, are better nowhere by 1%.
    const long long blocks = (p.m + 15) / 16, row_blocks = (p.rows + 15) / 16;
    if (row_blocks > 1 && blocks * row_blocks >= 512) launch_shrink<32, 2>(p, s);
    else launch_shrink<16, 4>(p, s);
    KCMM_HIP_CHECK(hipGetLastError(), err);
    if (p.rank <= 16) launch_expand_any<8, 1>(p, s);
    else if (p.rank <= 32) launch_expand_any<8, 2>(p, s);
    else if (p.rank <= 64) launch_expand_any<4, 4>(p, s);
    else launch_expand_any<4, 8>(p, s);
    KCMM_HIP_CHECK(hipGetLastError(), err);
    return true;
}

}  // namespace dev
}  // namespace kcmm
