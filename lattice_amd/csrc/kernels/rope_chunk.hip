// Rotation of a chunk's q and k, and the append of its k and v to the pages, for
// packed sequences of any lengths (gfx950).
//
// Row t of qkv holds [q heads | k heads | v heads] x D of one token.  Pair i of a
// rotated head (elements i and i + D/2) turns by the angle p * inv_freq[i]:
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin,
// p the token's place in the cache, or its position on the axis that pair i
// takes (time, height, width of an image's patches).  The angle is reduced in 64
// bits, in whole turns -- the product p * inv_freq / 2 pi of a 31-bit position has
// more bits than fp32, and a place of 10^5 would otherwise be off by 0.005 rad --
// so cos and sin are off by at most 2^-21 at places below 2^27 (2^-20 at any 32-bit
// position) with frequencies up to 1; each output is rounded once.
//
// Bound by HBM for prompts: each byte of qkv is read once, q and the page rows
// are written once; by its chain (the sequence of a token, its length, table
// entry, page offset) for a few tokens.
//  * Rows: a workgroup takes 4 tokens, their cosines and sines once into LDS
//    (64 pairs a token against 40 rotated heads), and a part of their heads; the
//    elements are loaded before the chain begins.
//  * fp8 pages: the rows that the chunk writes into a page have one scale per kv
//    head, so a wave takes one (page, kv head, K or V), or 2 or 4 waves do where the
//    page has more than they hold: rotated values stay in registers in 32 bits while
//    their maximum is found, and are encoded from there, without a rounding to bf16
//    between.  q heads are rows as above, in the same launch, behind the pages, whose
//    chain is longer (rows first: 35 for 32 us).  32 values a lane: with
//    64 the registers leave too few waves for the rows (32 for 26.6 us).
// Ragged prompts (32 q, 8 kv heads x 128): 4150 tokens 24 us in bf16, 4.2 TB/s
// read and written; 4507 into fp8 pages 24-26 us; 8 sequences of a few drafted tokens 7.4 us,
// a launch and the chain.
#include <algorithm>
#include <climits>
#include <cstring>

#include "../device_api.hpp"
#include "common.hpp"
#include "fp8_page.hpp"

namespace kcmm {
namespace {

struct ChunkParams {
    const uint8_t* qkv;
    uint8_t* q_out;
    uint8_t* k_base;
    uint8_t* v_base;
    const int32_t* block_tables;
    const int32_t* seq_lens;
    const int32_t* qsl;
    const uint64_t* offsets_f16;
    const float* inv_freq;
    const int32_t* positions;   // [axes][total], or null: the places
    uint32_t axis_bits[8];      // two bits per pair
    int batch, total, num_q_heads, kv_heads, head_dim, block_size, mbps, row_bytes, data_bytes;
    uint32_t n_ids;
    const uint32_t* issued;     // in a graph: the ids issued by now; or null
    int page_wgs;               // workgroups of the pages, in front of the rows
    int page_waves;             // waves of a page, kv head and K or V: 1, 2, 4
    int row_parts;              // of a tile of tokens' heads
};

constexpr int kTokens = 4;      // of a workgroup of rows (a wave finds each)
constexpr int kUnits = 2;       // 8-pair pieces of a thread

// cos and sin of p * f, p any 32-bit integer: whole turns are dropped in 64 bits
// (two roundings of 2^-53 of fewer than 2^29 turns; the rest is rounded to 2^-26).
__device__ __forceinline__ void turn(int p, float f, float* c, float* s) {
    const double turns = static_cast<double>(p) * static_cast<double>(f) * 0.15915494309189535;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), s, c);
}

__device__ __forceinline__ int axis_of(const ChunkParams& p, int pair) {
    return (p.axis_bits[pair >> 4] >> (2 * (pair & 15))) & 3;
}

// First place and end of sequence b's chunk in the cache, clamped to what its
// table holds (lo >= hi: nothing of it lies there).
struct Places {
    int first, lo, hi;
};
__device__ __forceinline__ Places places_of(const ChunkParams& p, int b) {
    const int q0 = p.qsl[b], q1 = p.qsl[b + 1], L = p.seq_lens[b];
    const long long cap = static_cast<long long>(p.mbps) * p.block_size;
    Places r;
    r.first = L - (q1 - q0);
    r.lo = max(r.first, 0);
    r.hi = static_cast<int>(min(static_cast<long long>(L), cap));
    if (q0 < 0 || q1 > p.total || q1 <= q0) r.hi = r.lo;
    return r;
}

// Block id of a sequence's block, or -1 for one that the pool has not issued.  A graph
// runs when the pool may have issued more ids than at its capture: their number is read
// from host memory, only for an id that was none then.
__device__ __forceinline__ int block_id(const ChunkParams& p, int b, int block) {
    const int32_t id = p.block_tables[static_cast<size_t>(b) * p.mbps + block];
    if (static_cast<uint32_t>(id) < p.n_ids) return id;
    if (p.issued == nullptr || id < 0) return -1;
    return static_cast<uint32_t>(id) < __hip_atomic_load(p.issued, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM) ? id : -1;
}

// C pairs of a row: elements e .. e+C-1 and e + D/2 .. of a head.
template <int DT, int C>
struct Pairs {
    static constexpr int W = C * io_bytes<DT>() / 4;   // dwords of each half
    uint32_t a[W], b[W];
    __device__ __forceinline__ void load(const uint8_t* at, int half) {
        half *= io_bytes<DT>();
        if constexpr (W % 4 == 0) {
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(at + 16 * i);
                const u32x4 y = *reinterpret_cast<const u32x4*>(at + half + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    a[4 * i + j] = x[j];
                    b[4 * i + j] = y[j];
                }
            }
        } else {
            const u32x2 x = *reinterpret_cast<const u32x2*>(at);
            const u32x2 y = *reinterpret_cast<const u32x2*>(at + half);
            a[0] = x[0];
            a[1] = x[1];
            b[0] = y[0];
            b[1] = y[1];
        }
    }
    __device__ __forceinline__ void store(uint8_t* at, int half) const {
        half *= io_bytes<DT>();
        if constexpr (W % 4 == 0) {
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
                *reinterpret_cast<u32x4*>(at + 16 * i) =
                    u32x4{a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]};
                *reinterpret_cast<u32x4*>(at + half + 16 * i) =
                    u32x4{b[4 * i], b[4 * i + 1], b[4 * i + 2], b[4 * i + 3]};
            }
        } else {
            *reinterpret_cast<u32x2*>(at) = u32x2{a[0], a[1]};
            *reinterpret_cast<u32x2*>(at + half) = u32x2{b[0], b[1]};
        }
    }
    __device__ __forceinline__ static float get(const uint32_t (&w)[W], int i) {
        if constexpr (DT == kDtF32) return __uint_as_float(w[i]);
        else return elem_to_f32<DT>(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu);
    }
    __device__ __forceinline__ void values(float (&x1)[C], float (&x2)[C]) const {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            x1[i] = get(a, i);
            x2[i] = get(b, i);
        }
    }
    __device__ __forceinline__ void set(const float (&y1)[C], const float (&y2)[C]) {
        if constexpr (DT == kDtF32) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                a[i] = __float_as_uint(y1[i]);
                b[i] = __float_as_uint(y2[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < C / 2; ++i) {
                a[i] = f32_to_elem<DT>(y1[2 * i]) | f32_to_elem<DT>(y1[2 * i + 1]) << 16;
                b[i] = f32_to_elem<DT>(y2[2 * i]) | f32_to_elem<DT>(y2[2 * i + 1]) << 16;
            }
        }
    }
};

// Rows: tokens wg / parts * kTokens .. and a part of their heads (Q_ONLY: the q
// heads; k and v go through page_waves).
template <int DT, int C, bool Q_ONLY>
__device__ __forceinline__ void rows(const ChunkParams& p, int wg) {
    constexpr int IO = DT == kDtFP8 ? kDtBF16 : DT;   // type of qkv and q
    __shared__ float2 s_turn[kTokens][128];           // cos, sin of a token's pairs
    __shared__ uint64_t s_row[kTokens];               // its page row, ~0: none
    __shared__ int s_place[kTokens];                  // -1: the token is skipped
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int D = p.head_dim, half = D / 2, per = half / C;
    const int Hq = p.num_q_heads, all = Hq + 2 * p.kv_heads, heads = Q_ONLY ? Hq : all;
    const int t0 = wg / p.row_parts * kTokens, part = wg % p.row_parts;
    const int units = kTokens * heads * per;
    Pairs<IO, C> x[kUnits];
    int head[kUnits], token[kUnits], piece[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int u = (part * kUnits + i) * 256 + tid;
        piece[i] = u % per;
        head[i] = u / per % heads;
        token[i] = u < units ? u / per / heads : -1;
        if (token[i] < 0 || t0 + token[i] >= p.total) {
            token[i] = -1;
            continue;
        }
        x[i].load(p.qkv + ((static_cast<size_t>(t0 + token[i]) * all + head[i]) * D + piece[i] * C) *
                              io_bytes<IO>(),
                  half);
    }
    if (wave < kTokens) {
        const int t = t0 + wave;
        int b = -1;
        for (int c = 0; c < p.batch && b < 0; c += 64) {
            const int i = min(c + lane, p.batch - 1);
            const unsigned long long hit = __ballot(p.qsl[i] <= t && t < p.qsl[i + 1]);
            if (hit) b = min(c + __ffsll(static_cast<long long>(hit)) - 1, p.batch - 1);
        }
        int place = -1;
        uint64_t row = ~0ull;
        if (b >= 0 && t < p.total) {
            const Places at = places_of(p, b);
            place = at.first + (t - p.qsl[b]);
            if (place < at.lo || place >= at.hi) place = -1;
            if (!Q_ONLY && place >= 0) {
                const int block = place / p.block_size, id = block_id(p, b, block);
                if (id >= 0)
                    row = p.offsets_f16[id] * 2ull +
                          static_cast<uint64_t>(place - block * p.block_size) * p.row_bytes;
            }
        }
        if (lane == 0) {
            s_place[wave] = place;
            s_row[wave] = row;
        }
    }
    __syncthreads();
    for (int i = tid; i < kTokens * half; i += 256) {
        const int t = i / half, pair = i - t * half;
        int at = s_place[t];
        if (at < 0) continue;
        if (p.positions != nullptr)
            at = p.positions[static_cast<size_t>(axis_of(p, pair)) * p.total + t0 + t];
        float2 cs;
        turn(at, p.inv_freq[pair], &cs.x, &cs.y);
        s_turn[t][pair] = cs;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        if (token[i] < 0 || s_place[token[i]] < 0) continue;
        const int h = head[i];
        uint8_t* dst;
        if (h < Hq) {
            dst = p.q_out + (static_cast<size_t>(t0 + token[i]) * Hq + h) * D * io_bytes<IO>();
        } else {
            const uint64_t row = s_row[token[i]];
            if (row == ~0ull) continue;
            const bool is_v = h >= Hq + p.kv_heads;
            dst = (is_v ? p.v_base : p.k_base) + row +
                  static_cast<size_t>(h - Hq - (is_v ? p.kv_heads : 0)) * D * io_bytes<IO>();
        }
        if (h < Hq + p.kv_heads) {
            float x1[C], x2[C], y1[C], y2[C];
            x[i].values(x1, x2);
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const float2 cs = s_turn[token[i]][piece[i] * C + j];
                y1[j] = rope_first(x1[j], x2[j], cs.x, cs.y);
                y2[j] = rope_second(x1[j], x2[j], cs.x, cs.y);
            }
            x[i].set(y1, y2);
        }
        x[i].store(dst + piece[i] * C * io_bytes<IO>(), half);
    }
}

// C values / scale as e4m3 codes.
template <int C>
__device__ __forceinline__ void put_codes(uint8_t* at, const float (&v)[C], float scale, float r,
                                          bool fast) {
    uint32_t w[C / 4];
#pragma unroll
    for (int i = 0; i < C / 4; ++i) {
        if (fast) {
            const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_quotient(v[4 * i], scale, r),
                                                           fp8_quotient(v[4 * i + 1], scale, r), 0, false);
            w[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(
                fp8_quotient(v[4 * i + 2], scale, r), fp8_quotient(v[4 * i + 3], scale, r), lo, true));
        } else {
            w[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i] |= f32_to_fp8e4m3(v[4 * i + j] / scale) << (8 * j);
        }
    }
    if constexpr (C == 8) *reinterpret_cast<u32x2*>(at) = u32x2{w[0], w[1]};
    else *reinterpret_cast<uint32_t*>(at) = w[0];
}

// `waves` waves of a workgroup: the chunk's rows of one (page, kv head, K or V), job =
// unit * 2 Hkv + 2 kvh + is_v over the pages that the sequences' chunks touch, in
// order.  The scale: as fp8_write_page_head has it.
template <int C>
__device__ __forceinline__ void page_waves(const ChunkParams& p, int wg) {
    __shared__ float s_amax[4];
    const int lane = threadIdx.x & 63, W = p.page_waves;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int job = wg * (4 / W) + wave / W, sub = wave % W;
    const int unit = job / (2 * p.kv_heads), j = job - unit * 2 * p.kv_heads;
    const int kvh = j >> 1;
    const bool is_v = j & 1;
    // the sequence and block of this unit
    int b = -1, block = 0, base = 0;
    for (int c = 0; c < p.batch && b < 0; c += 64) {
        int n = 0, b0 = 0;
        if (c + lane < p.batch) {
            const Places at = places_of(p, c + lane);
            b0 = at.lo / p.block_size;
            n = at.hi > at.lo ? (at.hi - 1) / p.block_size - b0 + 1 : 0;
        }
        int end = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(end, o);
            if (lane >= o) end += y;
        }
        const unsigned long long hit = __ballot(base + end > unit);
        if (hit) {
            const int at = __ffsll(static_cast<long long>(hit)) - 1;
            b = c + at;
            block = __shfl(b0, at) + unit - (base + __shfl(end - n, at));
        }
        base += __shfl(end, 63);
    }
    int id = b < 0 ? -1 : block_id(p, b, block);
    if (id < 0 && W == 1) return;
    const bool none = id < 0;   // (its waves go on to the barrier)
    if (none) b = block = id = 0;
    const Places at = places_of(p, b);
    const int D = p.head_dim, half = D / 2, per = half / C;
    const int s0 = max(at.lo - block * p.block_size, 0);
    const int s1 = none ? s0 : min(at.hi - block * p.block_size, p.block_size);
    // token of slot 0 (a row of qkv), place of slot 0
    const int place0 = block * p.block_size, tok0 = p.qsl[b] + place0 - at.first;
    const int all = p.num_q_heads + 2 * p.kv_heads;
    const int head = p.num_q_heads + (is_v ? p.kv_heads : 0) + kvh;
    uint8_t* page = (is_v ? p.v_base : p.k_base) + p.offsets_f16[id] * 2ull;
    float* const scale_at = reinterpret_cast<float*>(page + p.data_bytes) + kvh;
    const float old = none ? 0.0f : *scale_at;

    constexpr int PASS = 16 / C;        // pieces of a lane held at a time (32 values)
    const int pieces = (s1 - s0) * per, mine = sub * 64 * PASS, step = W * 64 * PASS;
    float y1[PASS][C], y2[PASS][C];
    bool nan = false;
    float amax = 0.0f;
    auto take = [&](int q0) {
        Pairs<kDtBF16, C> x[PASS];
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            const int q = min(q0 + i * 64 + lane, pieces - 1), s = s0 + q / per;
            x[i].load(p.qkv + ((static_cast<size_t>(tok0 + s) * all + head) * D + q % per * C) * 2, half);
        }
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            if (q0 + i * 64 >= pieces) break;   // (uniform)
            x[i].values(y1[i], y2[i]);
            if (is_v) continue;
            const int q = min(q0 + i * 64 + lane, pieces - 1), s = s0 + q / per;
#pragma unroll
            for (int k = 0; k < C; ++k) {
                const int pair = q % per * C + k;
                const int pos = p.positions == nullptr
                                    ? place0 + s
                                    : p.positions[static_cast<size_t>(axis_of(p, pair)) * p.total + tok0 + s];
                float cs, sn;
                turn(pos, p.inv_freq[pair], &cs, &sn);
                const float a = y1[i][k], c = y2[i][k];
                y1[i][k] = rope_first(a, c, cs, sn);
                y2[i][k] = rope_second(a, c, cs, sn);
            }
        }
    };
    for (int q0 = mine; q0 < pieces; q0 += step) {
        take(q0);
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            if (q0 + i * 64 >= pieces) break;   // (lanes past the end repeat the last piece)
#pragma unroll
            for (int k = 0; k < C; ++k) {
                amax = fmaxf(amax, fmaxf(fabsf(y1[i][k]), fabsf(y2[i][k])));
                nan |= __builtin_isunordered(y1[i][k], y2[i][k]);
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if (W > 1) {
        if (lane == 0) s_amax[wave] = amax;
        __syncthreads();
        for (int i = 0; i < W; ++i) amax = fmaxf(amax, s_amax[wave - sub + i]);
        if (none) return;
    }
    const bool fresh = s0 == 0 || !(old > 0.0f && old <= 3.40282347e38f);
    float scale = old;
    if (fresh) {
        scale = amax > 0.0f ? amax / 448.0f : 1.0f;
    } else if (amax > 448.0f * old) {
        scale = amax / 448.0f;
        // the slots that the chunk does not write, from the old scale to the new
        const int words = D / 8, rest = p.block_size - (s1 - s0);
        for (int q = sub * 64 + lane; q < rest * words; q += W * 64) {
            int s = q / words;
            if (s >= s0) s += s1 - s0;
            u32x2* const w = reinterpret_cast<u32x2*>(page + static_cast<size_t>(s) * p.row_bytes +
                                                      static_cast<size_t>(kvh) * D + q % words * 8);
            u32x2 v = *w;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t o = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    o |= f32_to_fp8e4m3(fp8e4m3_to_f32((v[i] >> (8 * k)) & 0xffu) * old / scale) << (8 * k);
                v[i] = o;
            }
            *w = v;
        }
    }
    const bool fast = !__any(nan) && scale >= kFp8QuotientMin && scale <= kFp8QuotientMax;
    const float r = 1.0f / scale;
    for (int q0 = mine; q0 < pieces; q0 += step) {
        if (pieces > step) take(q0);
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            const int q = q0 + i * 64 + lane;
            if (q >= pieces) continue;
            uint8_t* row = page + static_cast<size_t>(s0 + q / per) * p.row_bytes +
                           static_cast<size_t>(kvh) * D + q % per * C;
            put_codes<C>(row, y1[i], scale, r, fast);
            put_codes<C>(row + half, y2[i], scale, r, fast);
        }
    }
    if (sub == 0 && lane == 0) *scale_at = scale;
}

template <int DT, int C>
__global__ __launch_bounds__(256) void rope_chunk(ChunkParams p) {
    const int wg = static_cast<int>(blockIdx.x);
    if constexpr (DT == kDtFP8) {
        if (wg < p.page_wgs) {
            page_waves<C>(p, wg);
            return;
        }
    }
    rows<DT, C, DT == kDtFP8>(p, wg - p.page_wgs);
}

template <int DT>
bool launch_chunk(ChunkParams& p, hipStream_t s, std::string* err) {
    // pieces of 8 pairs where both halves of a head split into them (fp32: 4)
    const int C = DT != kDtF32 && p.head_dim % 16 == 0 ? 8 : 4;
    const long long heads = DT == kDtFP8 ? p.num_q_heads : p.num_q_heads + 2 * p.kv_heads;
    const long long units = kTokens * heads * (p.head_dim / 2 / C);
    const long long parts = (units + 256 * kUnits - 1) / (256 * kUnits);
    const long long tiles = (static_cast<long long>(p.total) + kTokens - 1) / kTokens;
    long long wgs = tiles * parts, page_wgs = 0;
    if (DT == kDtFP8) {
        // a chunk of n tokens touches at most (n - 1) / block_size + 2 pages
        const long long seqs = std::min(p.batch, p.total);
        const long long pages = std::min<long long>(p.total, (p.total - seqs) / p.block_size + 2 * seqs);
        // a wave for every 128 pieces of a full page, which it holds
        const int pieces = p.block_size * (p.head_dim / 2 / C), each = 64 * (16 / C);
        p.page_waves = pieces <= each ? 1 : pieces <= 2 * each ? 2 : 4;
        page_wgs = (pages * 2 * p.kv_heads * p.page_waves + 3) / 4;
    }
    if (wgs + page_wgs > INT_MAX) {
        *err = "too many tokens x heads";
        return false;
    }
    p.row_parts = static_cast<int>(parts);
    p.page_wgs = static_cast<int>(page_wgs);
    const dim3 grid(static_cast<unsigned>(wgs + page_wgs));
    if (C == 8) hipLaunchKernelGGL((rope_chunk<DT, DT == kDtF32 ? 4 : 8>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((rope_chunk<DT, 4>), grid, dim3(256), 0, s, p);
    KCMM_HIP_CHECK(hipGetLastError(), err);
    return true;
}

}  // namespace

namespace dev {

bool rope_append_chunk(const RopeChunkArgs& a, std::string* err) {
    if (a.total_query_tokens == 0) return true;
    ChunkParams p{};
    p.qkv = reinterpret_cast<const uint8_t*>(a.qkv);
    p.q_out = reinterpret_cast<uint8_t*>(a.q_out);
    p.k_base = reinterpret_cast<uint8_t*>(a.k_base);
    p.v_base = reinterpret_cast<uint8_t*>(a.v_base);
    p.block_tables = reinterpret_cast<const int32_t*>(a.block_tables);
    p.seq_lens = reinterpret_cast<const int32_t*>(a.seq_lens);
    p.qsl = reinterpret_cast<const int32_t*>(a.query_start_loc);
    p.offsets_f16 = reinterpret_cast<const uint64_t*>(a.offsets_f16);
    p.inv_freq = reinterpret_cast<const float*>(a.inv_freq);
    p.positions = reinterpret_cast<const int32_t*>(a.positions);
    for (uint32_t i = 0; i < a.head_dim / 2; ++i)
        p.axis_bits[i >> 4] |= static_cast<uint32_t>(a.axis_of_pair[i] & 3) << (2 * (i & 15));
    p.batch = static_cast<int>(a.batch);
    p.total = static_cast<int>(a.total_query_tokens);
    p.num_q_heads = static_cast<int>(a.num_q_heads);
    p.kv_heads = static_cast<int>(a.kv_heads);
    p.head_dim = static_cast<int>(a.head_dim);
    p.block_size = static_cast<int>(a.block_size);
    p.mbps = static_cast<int>(a.mbps);
    p.row_bytes = static_cast<int>(a.row_bytes);
    p.data_bytes = static_cast<int>(a.data_bytes);
    p.n_ids = a.n_ids;
    hipStream_t s = reinterpret_cast<hipStream_t>(a.stream);
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (s != nullptr && hipStreamIsCapturing(s, &capture) != hipSuccess)
        (void)hipGetLastError();   // (a stream that is never captured, while another one is)
    if (capture != hipStreamCaptureStatusNone) p.issued = reinterpret_cast<const uint32_t*>(a.issued_word);
    switch (a.dtype) {
        case kDtF16: return launch_chunk<kDtF16>(p, s, err);
        case kDtBF16: return launch_chunk<kDtBF16>(p, s, err);
        case kDtF32: return launch_chunk<kDtF32>(p, s, err);
        default: return launch_chunk<kDtFP8>(p, s, err);
    }
}

}  // namespace dev
}  // namespace kcmm
