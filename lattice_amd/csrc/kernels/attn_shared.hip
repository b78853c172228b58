// Paged decode attention of groups of sequences that share a prefix (gfx950).
//
//   out[b][h] = sum_t softmax_t(scale q[b][h].K[t]) V[t],  t < L_b,
// the whole blocks among the first min(shared_lens[b], L_b) tokens of sequence b
// (s_b tokens) being those of the first sequence of its group, through whose
// table they are read; the rest is read through b's own table.  L_b <= 0 writes
// zeros.  Sums, maxima and outputs are fp32 up to the store.
//
// Bound by HBM: a page that a group shares is read once for several of its
// sequences, instead of once for each.
//  * An item is a run of sequences of one group with the tokens that they have in
//    common, or one sequence with the tokens behind those.  The 16 NCB columns of
//    the matrix products are (sequence of the item, query head) pairs, so a K/V byte
//    serves up to 64 query rows, as one of a single sequence serves G (query heads a
//    kv head).  No column of an item is masked: where its sequences share different
//    lengths, the cut that saves most reads (or the least length, where that is near) is
//    taken, and those that share less are left to read their tokens by themselves.
//  * The work is the list of 8 KiB tiles (16 or 32 tokens) of all (item, kv head),
//    common tokens first; every wave takes an equal, contiguous slice of it.  Two
//    tiles a wave, one on its way, by direct loads into LDS, and two waves a SIMD: one
//    wave with larger tiles has a quarter of its time without loads in flight.
//    Each workgroup works out items and slices for itself, from lengths and group
//    starts, in LDS (a kernel in front would cost more than that).
//  * S^T = K Q^T and O^T += V^T P^T on 16x16x32 matrix instructions, softmax with a
//    running maximum in the log2 domain; V is turned by the transposing LDS read,
//    through LDS of the wave's own (no barrier in the loop).
//  * Parts of a (sequence, head) -- slices of the common tokens, slices of the rest
//    -- are joined by their log-sum-exp in a second kernel.  The waves of a workgroup
//    that end in the same (item, kv head) make one part of theirs in LDS first.
// 64 sequences over one prompt of 2048 with 64 to 512 tokens of their own (32 q, 8 kv
// heads x 128, bf16): 35 us, 2.5 TB/s of what has to be read once; 32 requests of four
// beams over 1 to 8 thousand tokens, fp8 pages: 95 us, 3.5 TB/s.  The launch and the
// chain length, table, offset, page in front of the first tile are 6 us of each, the
// joining kernel 6 more.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "../device_api.hpp"
#include "attn_stream.hpp"
#include "common.hpp"
#include "wide_pipe.hpp"

namespace kcmm {
namespace {

struct SharedParams {
    const uint8_t* q;
    uint8_t* out;
    const uint8_t* k_base;
    const uint8_t* v_base;
    const int32_t* block_tables;
    const int32_t* seq_lens;
    const int32_t* shared_lens;
    const int32_t* group_starts;
    const uint64_t* offsets_f16;
    int batch, groups, num_q_heads, kv_heads, head_dim, block_size, mbps, row_bytes, data_bytes;
    float scale;
};

__device__ __forceinline__ int whole_blocks(int n, int bs) { return n > 0 ? n / bs * bs : 0; }

// The first sequence of b's group, or -1: b lies in none.  The last group start
// not behind b (starts ascend; empty groups have the start of the next).
__device__ __forceinline__ int leader_of(const SharedParams& p, int b, int lane) {
    int n = 0;
    for (int c = 0; c <= p.groups; c += 64) {
        const int i = c + lane;
        n += __popcll(__ballot(i <= p.groups && p.group_starts[min(i, p.groups)] <= b));
    }
    if (n == 0 || n > p.groups) return -1;
    return min(max(p.group_starts[n - 1], 0), p.batch - 1);
}

// Any shape (head_dim <= 256, any GQA map, any block size, every page type): a
// workgroup a (sequence, query head).  Lanes form teams of T (4 dims each), which
// take the positions in turn, four at a time, each with its own maximum, sum and
// outputs; these meet by shuffles, then in LDS.  The page offsets (and fp8
// scales) of kChunk positions are staged in LDS before they are walked.
constexpr int kThreads = 512, kChunk = 1024, kUnroll = 4;

// Where a running maximum begins: finite, so that scores of -inf in front of every
// other leave 0 (and no NaN), and tokens of such scores alone 0 / 0.
constexpr float kLowest = -3.402823466e38f;

template <int DT>
__global__ __launch_bounds__(kThreads) void attn_shared_generic(SharedParams p, int tlog2) {
    constexpr bool F8 = DT == kDtFP8;
    __shared__ uint64_t s_page[kChunk + 1];
    __shared__ float s_ks[F8 ? kChunk + 1 : 1], s_vs[F8 ? kChunk + 1 : 1];
    __shared__ float s_m[kThreads / 64], s_s[kThreads / 64];
    __shared__ float s_acc[kThreads / 64 * 256];
    const int b = static_cast<int>(blockIdx.x) / p.num_q_heads;
    const int h = static_cast<int>(blockIdx.x) - b * p.num_q_heads;
    const int kvh = static_cast<int>(static_cast<long long>(h) * p.kv_heads / p.num_q_heads);
    const int tid = threadIdx.x, D = p.head_dim;
    const int T = 1 << tlog2, teams = kThreads >> tlog2, team = tid >> tlog2;
    const int d0 = (tid & (T - 1)) * 4;
    const int L = static_cast<int>(min(static_cast<long long>(p.seq_lens[b]),
                                       static_cast<long long>(p.mbps) * p.block_size));
    const size_t io_off = (static_cast<size_t>(b) * p.num_q_heads + h) * D * io_bytes<DT>();
    if (L <= 0) {
        for (int d = tid; d < D; d += kThreads) io_store<DT>(p.out + io_off, d, 0.0f);
        return;
    }
    const int lead = leader_of(p, b, tid & 63);
    const int shared = lead < 0 ? 0 : whole_blocks(min(p.shared_lens[b], L), p.block_size);
    float qv[4], acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        qv[i] = d0 + i < D ? io_load<DT>(p.q + io_off, d0 + i) : 0.0f;
        acc[i] = 0.0f;
    }
    const uint64_t head_off = static_cast<uint64_t>(kvh) * D * kv_elem_bytes<DT>();
    auto load4 = [&](const uint8_t* row, float sc, float (&x)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = d0 + i;
            if (d >= D) x[i] = 0.0f;
            else if constexpr (DT == kDtF32) x[i] = reinterpret_cast<const float*>(row)[d];
            else if constexpr (F8) x[i] = fp8e4m3_to_f32(row[d]) * sc;
            else x[i] = elem_to_f32<DT>(reinterpret_cast<const uint16_t*>(row)[d]);
        }
    };
    float m = kLowest, s = 0.0f;
    for (int end = 0, c0 = 0; c0 < L; c0 = end) {
        // up to kChunk positions of one table
        const int32_t* table = p.block_tables + static_cast<size_t>(c0 < shared ? lead : b) * p.mbps;
        end = min(c0 < shared ? shared : L, c0 + kChunk);
        const int lb0 = c0 / p.block_size, nb = (end - 1) / p.block_size - lb0 + 1;
        __syncthreads();
        for (int i = tid; i < nb; i += kThreads) {
            const uint64_t page = p.offsets_f16[table[lb0 + i]] * 2ull;
            s_page[i] = page;
            if constexpr (F8) {
                s_ks[i] = *reinterpret_cast<const float*>(p.k_base + page + p.data_bytes + kvh * 4);
                s_vs[i] = *reinterpret_cast<const float*>(p.v_base + page + p.data_bytes + kvh * 4);
            }
        }
        __syncthreads();
        for (int pos = c0 + team; pos < end; pos += teams * kUnroll) {
            float kx[kUnroll][4], vx[kUnroll][4], dot[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int at = min(pos + u * teams, end - 1);
                const int lb = at / p.block_size, j = lb - lb0;
                const uint64_t row = s_page[j] + static_cast<uint64_t>(at - lb * p.block_size) * p.row_bytes +
                                     head_off;
                load4(p.k_base + row, F8 ? s_ks[j] : 1.0f, kx[u]);
                load4(p.v_base + row, F8 ? s_vs[j] : 1.0f, vx[u]);
            }
            float top = m;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                dot[u] = qv[0] * kx[u][0] + qv[1] * kx[u][1] + qv[2] * kx[u][2] + qv[3] * kx[u][3];
                for (int o = T >> 1; o > 0; o >>= 1) dot[u] += __shfl_xor(dot[u], o);
                dot[u] = pos + u * teams < end ? dot[u] * p.scale : -INFINITY;
                top = fmaxf(top, dot[u]);
            }
            const float corr = kexp<DT>(m - top);
            s *= corr;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] *= corr;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (pos + u * teams >= end) continue;
                const float e = kexp<DT>(dot[u] - top);
                s += e;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] += e * vx[u][i];
            }
            m = top;
        }
    }
    float M = m;
    for (int o = T; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
    const float f = kexp<DT>(m - M);
    s *= f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= f;
    for (int o = T; o < 64; o <<= 1) {
        s += __shfl_xor(s, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], o);
    }
    const int wave = tid >> 6;
    if ((tid & 63) < T)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_acc[wave * 256 + d0 + i] = acc[i];
    if ((tid & 63) == 0) {
        s_m[wave] = M;
        s_s[wave] = s;
    }
    __syncthreads();
    for (int d = tid; d < D; d += kThreads) {
        float top = kLowest, S = 0.0f, o = 0.0f;
        for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, s_m[w]);
        for (int w = 0; w < kThreads / 64; ++w) {
            const float e = kexp<DT>(s_m[w] - top);
            S += s_s[w] * e;
            o += s_acc[w * 256 + d] * e;
        }
        io_store<DT>(p.out + io_off, d, o / S);
    }
}

template <int DT>
void launch_generic(const SharedParams& p, hipStream_t s) {
    int tlog2 = 2;
    while ((4 << tlog2) < p.head_dim) ++tlog2;   // 4 T >= head_dim, T <= 64
    hipLaunchKernelGGL(attn_shared_generic<DT>, dim3(static_cast<unsigned>(p.batch) * p.num_q_heads),
                       dim3(kThreads), 0, s, p, tlog2);
}

// ---- whole GQA groups of at most 16 heads, head_dim 64 or 128, pages of 8-token groups ----

constexpr int kWaves = 4;              // of a workgroup
constexpr int kMaxRows = 64 * kWaves;   // sequences of a launch: one a thread in find_items

// What the joining kernel has to know of a sequence: where its parts are.
struct RowPlan {
    int pre_tile, pre_tiles;   // first tile of the item's common tokens (kv head 0), their number; 0: none
    int first;                 // first sequence of the item
    int own_tile, own_tiles;   // the same of the tokens behind them
};

struct FastParams {
    SharedParams p;
    int row0, rows;            // sequences of this launch
    int group, seqs;           // query heads a kv head; sequences of an item
    int slices;                // waves
    int* per;                  // tiles of a slice, of all, and common ones a kv head: for the joining kernel
    RowPlan* plan;
    // first parts of (sequence, head): of the common tokens, then of the rest;
    // later parts by slice, a row a column
    float *ml, *acc, *slice_ml, *slice_acc;
    float scale_log2;
};

// Tokens of a tile: 8 KiB of K and V, so that two tiles for each of eight waves fit
// the LDS of a CU.
constexpr int tile_tokens(int row_bytes) { return row_bytes == 256 ? 16 : 32; }
__device__ __forceinline__ int tiles_of(int tokens, int tile) { return (tokens + tile - 1) / tile; }

// The items of this launch, in LDS, by sequence (relative to row0).
struct Items {
    int len[kMaxRows];      // tokens, clamped to what the table holds
    int shared[kMaxRows];   // tokens in shared blocks
    int lead[kMaxRows];     // whose table these are read through (of the whole batch)
    int common[kMaxRows];   // tokens that the item of the sequence takes in common; 0: none
    int count[kMaxRows];    // sequences of the item that begins here, 0: none does
    int most[kMaxRows];     // the most and the least that one of them shares; then
    int least[kMaxRows];    // least: their common tokens
    unsigned long long best[kMaxRows];   // what the best cut saves, and that cut
    int pre[kMaxRows];      // tiles of the items before this sequence, of one kv head
    int own[kMaxRows];      // the same of the sequences' own tokens
    uint64_t begins[kWaves];   // bit of a wave's lane: a group begins there
    int sums[2][kWaves];
    int carry;
};

// Sum over lanes 0 .. l, by row shifts and row broadcasts.
__device__ __forceinline__ int wave_sums(int x) {
#define KCMM_ADD(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xF, false)
    KCMM_ADD(0x111, 0xF);   // row_shr:1, 2, 4, 8
    KCMM_ADD(0x112, 0xF);
    KCMM_ADD(0x114, 0xF);
    KCMM_ADD(0x118, 0xF);
    KCMM_ADD(0x142, 0xA);   // row_bcast:15 into rows 1 and 3
    KCMM_ADD(0x143, 0xC);   // row_bcast:31 into rows 2 and 3
#undef KCMM_ADD
    return x;
}

// One sequence a thread.  (Every workgroup spends this before its first load, so
// nothing walks over sequences: an item's members meet in LDS atomics.)
template <int TILE>
__device__ __forceinline__ void find_items(const FastParams& f, Items& it) {
    const SharedParams& p = f.p;
    const int r = threadIdx.x, lane = r & 63, wave = r >> 6, b = f.row0 + r;
    int len = 0, shared = 0;
    if (r < f.rows) {
        len = max(0, min(p.seq_lens[b], p.mbps * p.block_size));
        shared = p.shared_lens[b];
    }
    const int end = p.group_starts[p.groups];   // sequences from here on lie in no group
    it.len[r] = len;
    it.common[r] = it.count[r] = it.most[r] = 0;
    it.best[r] = 0;
    it.least[r] = INT_MAX;
    it.lead[r] = -1;
    if (r == 0) it.carry = -1;
    __syncthreads();
    for (int g = r; g < p.groups; g += kMaxRows) {
        const int start = p.group_starts[g];
        if (start < 0 || start >= f.row0 + f.rows) continue;
        if (start >= f.row0) it.lead[start - f.row0] = start;
        else atomicMax(&it.carry, start);
    }
    __syncthreads();
    const uint64_t mine = __ballot(it.lead[r] >= 0);
    if (lane == 0) it.begins[wave] = mine;
    __syncthreads();
    // the last group start not behind the sequence
    int lead = it.carry;
    for (int w = 0; w <= wave; ++w) {
        const uint64_t m = w < wave ? it.begins[w] : mine & (~0ull >> (63 - lane));
        if (m) lead = f.row0 + 64 * w + 63 - __clzll(static_cast<long long>(m));
    }
    const bool in = r < f.rows && lead >= 0 && b < end;
    shared = in ? whole_blocks(min(shared, len), p.block_size) : 0;
    it.shared[r] = shared;
    it.lead[r] = lead;
    // the sequence's item begins at `first`
    const int from = max(lead - f.row0, 0), first = from + (r - from) / f.seqs * f.seqs;
    if (in) {
        atomicMax(&it.most[first], shared);
        atomicMin(&it.least[first], shared);
        atomicAdd(&it.count[first], 1);
    }
    __syncthreads();
    // The common tokens: of the lengths that the item's sequences share, the c with the most
    // (k - 1) c saved, k of them sharing c or more (both in units of 8 tokens, below 2^34
    // and 2^28); the others read all of theirs by themselves.  Where all share nearly the
    // same it is the least: the search takes 1 to 2 us, and could save an eighth at most.
    const int count = in ? it.count[first] : 0, least = in ? it.least[first] : 0;
    const bool unequal = in && 8ll * least < 7ll * it.most[first];
    if (unequal && shared > 0) {
        int others = -1;
        for (int i = 0; i < count; ++i) others += it.shared[first + i] >= shared;
        const unsigned long long c = static_cast<unsigned>(shared) / 8;
        atomicMax(&it.best[first], others * c << 28 | (others > 0 ? c : 0));
    }
    __syncthreads();
    // (of one sequence alone there is nothing to gain)
    const int cut = unequal ? static_cast<int>(it.best[first] & 0xfffffff) * 8 : count > 1 ? least : 0;
    const int common = cut > 0 && shared >= cut ? cut : 0;
    const bool begins = in && first == r && cut > 0;
    const int pre = begins ? tiles_of(cut, TILE) : 0, own = tiles_of(len - common, TILE);
    it.common[r] = common;
    it.least[r] = cut;
    if (!begins) it.count[r] = 0;
    const int pre_to = wave_sums(pre), own_to = wave_sums(own);
    if (lane == 63) {
        it.sums[0][wave] = pre_to;
        it.sums[1][wave] = own_to;
    }
    __syncthreads();
    int before[2] = {0, 0};
    for (int w = 0; w < wave; ++w) {
        before[0] += it.sums[0][w];
        before[1] += it.sums[1][w];
    }
    it.pre[r] = before[0] + pre_to - pre;
    it.own[r] = before[1] + own_to - own;
    __syncthreads();
}

// Tiles of a slice: equal parts of all.
__device__ __forceinline__ int slice_tiles(int total, const FastParams& f) {
    return max((total + f.slices - 1) / f.slices, 1);
}

// LDS accesses of the streaming loop, at byte addresses and constant offsets, each
// block with its own wait.  Written out because the compiler, which cannot tell
// where in LDS a direct load will write, waits for all loads in flight before every
// LDS access that it makes itself.  A wave's LDS accesses are performed in order.
template <int O0, int O1>
__device__ __forceinline__ void lds_read(u32x4 (&x)[2][2], const uint32_t (&a)[2]) {
    asm volatile("ds_read_b128 %0, %4 offset:%6\n\tds_read_b128 %1, %5 offset:%6\n\t"
                 "ds_read_b128 %2, %4 offset:%7\n\tds_read_b128 %3, %5 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[1][0]), "=&v"(x[1][1])
                 : "v"(a[0]), "v"(a[1]), "i"(O0), "i"(O1) : "memory");
}
template <int O0, int>
__device__ __forceinline__ void lds_read(u32x4 (&x)[1][4], const uint32_t (&a)[4]) {
    asm volatile("ds_read_b128 %0, %4 offset:%8\n\tds_read_b128 %1, %5 offset:%8\n\t"
                 "ds_read_b128 %2, %6 offset:%8\n\tds_read_b128 %3, %7 offset:%8\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[0][2]), "=&v"(x[0][3])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(O0) : "memory");
}
// Transposing reads: of a 16-lane group, lane a + 4 s gives the address of four
// 16-bit elements M[a + 4 s][0 .. 3], lane 4 a + e receives M[a][e], M[a + 4][e],
// M[a + 8][e], M[a + 12][e].
template <int O0, int O1>
__device__ __forceinline__ void lds_read_turned(u32x2 (&x)[4][2], const uint32_t (&a)[4]) {
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[1][0]), "=&v"(x[1][1]), "=&v"(x[2][0]),
                   "=&v"(x[2][1]), "=&v"(x[3][0]), "=&v"(x[3][1])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(O0), "i"(O1) : "memory");
}
template <int O0, int>
__device__ __forceinline__ void lds_read_turned(u32x2 (&x)[4][1], const uint32_t (&a)[4]) {
    asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%8\n\tds_read_b64_tr_b16 %1, %5 offset:%8\n\t"
                 "ds_read_b64_tr_b16 %2, %6 offset:%8\n\tds_read_b64_tr_b16 %3, %7 offset:%8\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0][0]), "=&v"(x[1][0]), "=&v"(x[2][0]), "=&v"(x[3][0])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(O0) : "memory");
}
template <int O>
__device__ __forceinline__ void lds_write(uint32_t a, u32x4 x) {
    asm volatile("ds_write_b128 %0, %1 offset:%2" :: "v"(a), "v"(x), "i"(O) : "memory");
}
// Two fp32 -> one dword of 16-bit elements (round to nearest even).
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (DT == kDtF16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(lo), static_cast<_Float16>(hi)});
    } else {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(lo), static_cast<__bf16>(hi)});
    }
}
// What the elements of `packed` = pack2(lo, hi) leave of the values.
template <int DT>
__device__ __forceinline__ uint32_t pack2_rest(float lo, float hi, uint32_t packed) {
    return pack2<DT>(lo - elem_to_f32<DT>(packed & 0xffffu), hi - elem_to_f32<DT>(packed >> 16));
}
// Maximum over the lanes l, l ^ 16, l ^ 32, l ^ 48 that hold a column.
__device__ __forceinline__ float column_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// s_waitcnt vmcnt(N) (gfx9 encoding: vmcnt bits 3:0 and 15:14, the others at most).
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)p));
}

template <int DT, int D, int BS, int NCB>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2)))
void attn_shared_stream(FastParams f, const int32_t* __restrict__ bt, const uint64_t* __restrict__ offs,
                        const uint8_t* __restrict__ kreg, const uint8_t* __restrict__ vreg) {
    constexpr bool F8 = DT == kDtFP8;
    constexpr int MDT = F8 ? kDtBF16 : DT;     // matrix, q and out element type
    constexpr int EB = F8 ? 1 : 2;
    constexpr int KC = D / 32, DB = D / 16;
    constexpr int ROWB = D * EB;               // bytes of a token's head row
    constexpr int TILE = tile_tokens(ROWB), NH = TILE / 16;   // tokens of a tile, 16-token halves
    constexpr int GROUPS = TILE / 8;           // 8-token groups, each inside a page
    constexpr int HALF = TILE * ROWB;          // bytes of a tile's K, and of its V
    constexpr int LOADS = 2 * HALF / 1024;     // of a tile
    constexpr int ST = 2;                      // tiles of the ring
    static_assert(!F8 || D == 128, "fp8 pages take this path at head_dim 128");
    __shared__ Items it;
    __shared__ int s_key[kWaves], s_began[kWaves];
    __shared__ float2 s_ml[kWaves][NCB * 16];
    __shared__ __attribute__((aligned(1024))) uint8_t s_ring[kWaves][ST * 2 * HALF];
    const SharedParams& p = f.p;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int ln = lane & 15, lg = lane >> 4;
    const int bs = BS > 0 ? BS : p.block_size;
    const int Hkv = p.kv_heads, Hq = p.num_q_heads, G = f.group;
    auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };

    find_items<TILE>(f, it);
    int pre_all = 0, own_all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        pre_all += it.sums[0][w];
        own_all += it.sums[1][w];
    }
    const int pre_head = max(uni(pre_all), 1), pre_end = uni(pre_all) * Hkv, total = pre_end + uni(own_all) * Hkv;
    const int per = slice_tiles(total, f);
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) {
            f.per[0] = per;
            f.per[1] = total;
            f.per[2] = uni(pre_all);
        }
        const int r = threadIdx.x;
        if (r < f.rows) {
            RowPlan w{};
            w.own_tile = pre_end + it.own[r] * Hkv;
            w.own_tiles = tiles_of(it.len[r] - it.common[r], TILE);
            if (it.common[r] > 0) {
                const int from = max(it.lead[r] - f.row0, 0), first = from + (r - from) / f.seqs * f.seqs;
                w.first = f.row0 + first;
                w.pre_tile = it.pre[first];
                w.pre_tiles = tiles_of(it.common[r], TILE);
            }
            f.plan[r] = w;
        }
    }
    // The common tokens' tiles are listed by kv head, and an XCD (every eighth workgroup)
    // takes an eighth of them side by side: the items of a long prefix, which has more
    // sequences than one item holds, find its pages in that XCD's L2 (64 sequences of 4
    // heads over 2048 tokens, eight items: 40.6 -> 38.1 us).
    int wg = blockIdx.x;
    const int eighth = pre_end / (kWaves * per) / 8;
    if (wg < 8 * eighth) wg = wg % 8 * eighth + wg / 8;
    const int slice = wg * kWaves + wave;
    if (static_cast<long long>(wg) * kWaves * per >= total) return;   // (the whole workgroup)
    const int t0 = static_cast<int>(min(static_cast<long long>(slice) * per, static_cast<long long>(total)));
    const int n = min(per, total - t0);   // 0: nothing left for this wave

    // Cursor over the tile list: tokens begin + TILE t .. of (item, kv head); all of it
    // wave-uniform, so that the tables are read by scalar loads
    struct Cur {
        int r, own, g, t, nt, begin, end, shared, lead, seqs, blocks, again;
        float ks[F8 ? GROUPS : 1], vs[F8 ? GROUPS : 1];   // fp8: page scales of the 8-token groups
    };
    auto locate = [&](int tile) __attribute__((always_inline)) {
        Cur c;
        c.own = tile >= pre_end;
        const int* sums = c.own ? it.own : it.pre;
        // (own tokens by sequence, then kv head: a table's entries serve all its heads)
        const int rel = c.own ? tile - pre_end : tile % pre_head, x = c.own ? rel / Hkv : rel;
        // the last sequence with sums[r] <= x: it has tiles
        int lo = -1;
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            lo += __popcll(__ballot(sums[64 * w + lane] <= x && 64 * w + lane < f.rows));
        c.r = lo;
        c.seqs = c.own ? 1 : uni(it.count[lo]);
        c.blocks = (c.seqs * G + 15) >> 4;
        const int common = uni(c.own ? it.common[lo] : it.least[lo]);
        c.begin = c.own ? common : 0;
        c.end = c.own ? uni(it.len[lo]) : common;
        c.shared = c.own ? uni(it.shared[lo]) : common;
        c.lead = max(uni(it.lead[lo]), 0);
        c.nt = max(tiles_of(c.end - c.begin, TILE), 1);
        // whether another item reads these tokens too
        const int next = min(lo + max(c.seqs, 1), f.rows - 1);
        c.again = !c.own && ((lo > 0 && uni(it.lead[lo - 1]) == uni(it.lead[lo])) ||
                             (next > lo && uni(it.lead[next]) == uni(it.lead[lo]) && next == lo + c.seqs));
        const int rem = rel - uni(sums[lo]) * (c.own ? Hkv : 1);
        c.g = c.own ? rem / c.nt : tile / pre_head;
        c.t = c.own ? rem - c.g * c.nt : rem;
        return c;
    };
    Cur ic = locate(min(t0, total - 1));
    // (tile: the cursor's new place in the list)
    auto advance = [&](Cur& c, int tile) __attribute__((always_inline)) {
        if (++c.t < c.nt) return;
        c.t = 0;
        if (!c.own || ++c.g == Hkv) c = locate(tile);
    };
    // Byte offsets of 64 8-token groups' rows (512 tokens), a lane each, from tile
    // `from` of (sequence, kind) on; groups past the end repeat the last one
    // (masked).  They hold for every kv head.  What is loaded here is waited for at
    // once: a register that a load may still be on its way to would have every later
    // step wait for all loads in flight.
    struct {
        int r, own, from, g;
        uint64_t row;
        uint32_t slot;                   // of it, inside its page
        float ks, vs;                    // fp8: the groups' page scales of kv head g
    } pages;
    pages.r = -1;
    constexpr int AHEAD = 64 / GROUPS;   // tiles of these
    // Where the tile's groups lie for the tile's kv head (fp8: also their scales)
    auto group_bases = [&](Cur& c, uint64_t* gb) __attribute__((always_inline)) {
        bool fresh = false;
        if (pages.r != c.r || pages.own != c.own || c.t / AHEAD * AHEAD != pages.from) {
            pages.from = c.t / AHEAD * AHEAD;
            const int tok = c.begin + min(TILE * pages.from + 8 * lane, (c.end - 1 - c.begin) & ~7);
            const int row = tok < c.shared ? c.lead : f.row0 + c.r, block = tok / bs;
            const uint64_t page = offs[bt[static_cast<size_t>(row) * p.mbps + block]];
            pages.slot = static_cast<uint32_t>((tok - block * bs) * p.row_bytes);
            pages.row = page * 2ull + pages.slot;
            pages.r = c.r;
            pages.own = c.own;
            fresh = true;
        }
        if constexpr (F8) {
            if (fresh || pages.g != c.g) {
                const uint64_t at = pages.row - pages.slot + static_cast<uint32_t>(p.data_bytes + c.g * 4);
                pages.ks = *reinterpret_cast<const float*>(kreg + at);
                pages.vs = *reinterpret_cast<const float*>(vreg + at);
                pages.g = c.g;
                wait_loads<0>();
            }
        }
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) {
            const int j = min(GROUPS * c.t + q, (c.end - 1 - c.begin) >> 3) - GROUPS * pages.from;
            const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(pages.row), j);
            const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(pages.row >> 32), j);
            gb[q] = (static_cast<uint64_t>(hi) << 32 | lo) + static_cast<uint32_t>(c.g * D * EB);
            if constexpr (F8) {
                c.ks[q] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pages.ks), j));
                c.vs[q] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pages.vs), j));
            }
        }
    };
    // A tile's rows lie in the ring one behind the other, 16-byte piece x of row r at
    // x ^ (r & 15), or x ^ (r / 2 & 7) for rows of 128 bytes: then the 16 rows of a
    // matrix operand, and those of a transposing read, are in 16 places of the 64
    // banks.  A load instruction brings 1024 bytes: 4 rows or 8.
    constexpr int PIECES = ROWB / 16, ROWS = 64 / PIECES;
    auto turned = [](int row, int piece) __attribute__((always_inline)) {
        return row * ROWB + (ROWB == 256 ? piece ^ (row & 15) : piece ^ (row >> 1 & 7)) * 16;
    };
    uint8_t* const ring = s_ring[wave];
    constexpr int STEP = 16 / ROWS;   // loads after which the rows' pieces repeat
    uint32_t src[STEP];               // this lane's byte of an 8-token group, of load i % STEP
#pragma unroll
    for (int i = 0; i < STEP; ++i) {
        const int row = i * ROWS + lane / PIECES;
        const int piece = ROWB == 256 ? (lane % PIECES) ^ (row & 15) : (lane % PIECES) ^ (row >> 1 & 7);
        src[i] = static_cast<uint32_t>((row & 7) * p.row_bytes + piece * 16);
    }
    // (What is read once does not push out of the caches what is not: 332 MB of beams'
    // pages take 95 us so and 100 without; a prompt of eight items 35 us with its pages
    // left in the caches, 38 without.)
    auto issue = [&](uint32_t place, const uint64_t* gb, bool again) __attribute__((always_inline)) {
        uint8_t* const to = ring + place;
        if (again) {
#pragma unroll
            for (int i = 0; i < TILE / ROWS; ++i) {
                const uint64_t g = gb[i * ROWS / 8];
                load_lds16(kreg + g + src[i % STEP], to + i * 1024);
                load_lds16(vreg + g + src[i % STEP], to + HALF + i * 1024);
            }
        } else {
#pragma unroll
            for (int i = 0; i < TILE / ROWS; ++i) {
                const uint64_t g = gb[i * ROWS / 8];
                load_lds16_nt(kreg + g + src[i % STEP], to + i * 1024);
                load_lds16_nt(vreg + g + src[i % STEP], to + HALF + i * 1024);
            }
        }
    };
    // Column c of an item: head c % G of the kv head's, of its sequence c / G.
    // Columns past the last repeat one; they are computed and never stored.
    int seq_of[NCB], head_of[NCB];
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
        seq_of[cb] = (cb * 16 + ln) / G;
        head_of[cb] = cb * 16 + ln - seq_of[cb] * G;
    }
    u32x4 qf[NCB][KC];
    auto load_q = [&](const Cur& c) __attribute__((always_inline)) {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            const int row = f.row0 + c.r + min(seq_of[cb], c.seqs - 1);
            const uint8_t* qrow = p.q + (static_cast<size_t>(row) * Hq + c.g * G + head_of[cb]) * D * 2;
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) {
                const int e0 = F8 ? (kc >> 1) * 64 + (kc & 1) * 8 + 16 * lg : kc * 32 + lg * 8;
                qf[cb][kc] = *reinterpret_cast<const u32x4*>(qrow + e0 * 2);
            }
        }
    };

    float m_run[NCB], l_run[NCB];
    f32x4 acc[NCB][DB];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            m_run[cb] = kLowest;
            l_run[cb] = 0.0f;
#pragma unroll
            for (int i = 0; i < DB; ++i) acc[cb][i] = f32x4{0, 0, 0, 0};
        }
    };
    clear();

    // Where a part's outputs and its (maximum, sum) go: the part where a (sequence,
    // head) begins has a row of its own; later ones have the slice's place, in the
    // order of the registers, which makes whole lines of the stores.
    auto part_acc = [&](const Cur& c, bool begins, int slice, int cb) __attribute__((always_inline)) {
        const int row = (c.own * f.rows + c.r + seq_of[cb]) * Hq + c.g * G + head_of[cb];
        return begins ? f.acc + static_cast<size_t>(row) * D + 4 * lg
                      : f.slice_acc + static_cast<size_t>(slice * NCB + cb) * (16 * D) + lane * 4;
    };
    auto part_ml = [&](const Cur& c, bool begins, int slice, int cb) __attribute__((always_inline)) {
        const int row = (c.own * f.rows + c.r + seq_of[cb]) * Hq + c.g * G + head_of[cb];
        return reinterpret_cast<float2*>(begins ? f.ml : f.slice_ml) + (begins ? row : (slice * NCB + cb) * 16 + ln);
    };
    auto flush = [&](const Cur& c, bool begins) __attribute__((always_inline)) {
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            if (cb >= c.blocks) break;
            const float l = wave_sum_across_groups(l_run[cb]);
            if (seq_of[cb] >= c.seqs) continue;
            float* const to = part_acc(c, begins, slice, cb);
            const int step = begins ? 16 : 256;
#pragma unroll
            for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(to + db * step) = acc[cb][db];
            if (lg == 0) *part_ml(c, begins, slice, cb) = float2{m_run[cb], l};
        }
        clear();
    };

    // this lane's places in a tile: pieces of K's operand rows, of V's transposed ones,
    // and where it writes V's (fp8: as bf16, in padded rows)
    constexpr int NP = F8 ? KC / 2 : KC;
    const uint32_t at0 = lds_address(ring);
    const uint32_t k_at = at0 + turned(ln, lg);   // piece 4 i + lg: 64 i bytes of the turn
    // (V's rows as they are read: 2 D bytes, turned as rows of that length are)
    auto v_turned = [](int row, int piece) __attribute__((always_inline)) {
        return row * 2 * D + (D == 128 ? piece ^ (row & 15) : piece ^ (row >> 1 & 7)) * 16;
    };
    // (block db: 32 db bytes of the turn)
    const uint32_t v_at = at0 + v_turned(4 * lg + (ln >> 2), (ln & 3) >> 1) + (ln & 1) * 8;
    auto compute = [&](uint32_t place, const Cur& c) __attribute__((always_inline)) {
        constexpr int TK = 0, TV = HALF;
        const int tbase = c.begin + c.t * TILE;
        // rows past the end may hold anything and become zeros
        if (tbase + TILE > c.end)
            for (int row = c.end - tbase + lane / PIECES; row < TILE; row += ROWS)
                lds_write<TV>(at0 + place + row * ROWB + lane % PIECES * 16, u32x4{0, 0, 0, 0});
        uint32_t kp[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) kp[i] = (k_at + place) ^ (64 * i);
        u32x4 x[NH][NP];
        lds_read<TK, TK + 16 * ROWB>(x, kp);
        if constexpr (F8) {
            // V as bf16 (exactly: the pages' scales go to P), over the tile's K and V
            u32x4 y[2][NP];
            lds_read<TV, TV + 16 * ROWB>(y, kp);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = 16 * h + ln, piece = 2 * (4 * e + lg);
                    lds_write<0>(at0 + place + v_turned(row, piece), fp8x8_to_bf16(y[h][e][0], y[h][e][1]));
                    lds_write<0>(at0 + place + v_turned(row, piece + 1), fp8x8_to_bf16(y[h][e][2], y[h][e][3]));
                }
        }
        u32x4 pf[NCB][NH];
        const bool live = tbase + TILE <= c.end;   // (uniform)
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            if (cb >= c.blocks) break;   // (uniform: no column of the item lies here)
            f32x4 s[NH];
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                s[h] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    u32x4 a = x[h][F8 ? kc >> 1 : kc];
                    if constexpr (F8) a = (kc & 1) ? fp8x8_to_bf16(a[2], a[3]) : fp8x8_to_bf16(a[0], a[1]);
                    s[h] = mfma16x16x32<MDT>(a, qf[cb][kc], s[h]);
                }
            }
            float v[4 * NH], sum = 0.0f;
            float mt = -INFINITY;
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                float sc = f.scale_log2;
                if constexpr (F8) sc *= lg < 2 ? c.ks[2 * h] : c.ks[2 * h + 1];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float z = s[h][r] * sc;
                    v[h * 4 + r] = live || tbase + h * 16 + lg * 4 + r < c.end ? z : -INFINITY;
                    mt = fmaxf(mt, v[h * 4 + r]);
                }
            }
            // the column's reference grows where a score exceeds it by more than 8: until
            // then weights are at most 2^8 of the greatest, which costs no bits.  f16 weights
            // are 2^7 times as large, up to 2^15: below 2^-25 f16 has nothing, and a tile of
            // weights of 2^-26 beside one of 1 would be lost
            constexpr float UP = DT == kDtF16 ? 7.0f : 0.0f;
            if (__any(mt > m_run[cb] + (8.0f + UP))) {
                const float m_new = fmaxf(m_run[cb], column_max(mt) - UP);
                const float corr = __builtin_amdgcn_exp2f(m_run[cb] - m_new);
                l_run[cb] *= corr;
                m_run[cb] = m_new;
#pragma unroll
                for (int i = 0; i < DB; ++i) acc[cb][i] *= corr;
            }
#pragma unroll
            for (int i = 0; i < 4 * NH; ++i) {
                v[i] = __builtin_amdgcn_exp2f(v[i] - m_run[cb]);
                sum += v[i];
            }
            l_run[cb] += sum;
            if constexpr (F8) {
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const float vs = lg < 2 ? c.vs[2 * h] : c.vs[2 * h + 1];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[h * 4 + r] *= vs;
                }
            }
            // slots (lg, i) of a half's P^T operand: token 4 lg + i % 4, its weight and what
            // that leaves (one part alone, 2^-9 of a weight, would be as large an error as
            // the store's; 16 tokens would leave half the slots empty anyway)
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                const float* w = v + 4 * h;
                const uint32_t a = pack2<MDT>(w[0], w[1]), b = pack2<MDT>(w[2], w[3]);
                pf[cb][h] = u32x4{a, b, pack2_rest<MDT>(w[0], w[1], a), pack2_rest<MDT>(w[2], w[3], b)};
            }
        }
#pragma unroll
        for (int d0 = 0; d0 < DB; d0 += 4) {
            // lane (ln, lg): V[4 lg .. +3][16 db + ln], and of the second half
            u32x2 t[4][NH];
            const uint32_t v0 = v_at + place;
            const uint32_t at[4] = {v0 ^ 32 * d0, v0 ^ 32 * (d0 + 1), v0 ^ 32 * (d0 + 2), v0 ^ 32 * (d0 + 3)};
            lds_read_turned<F8 ? 0 : TV, (F8 ? 0 : TV) + 32 * D>(t, at);
#pragma unroll
            for (int cb = 0; cb < NCB; ++cb) {
                if (cb >= c.blocks) break;
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int h = 0; h < NH; ++h)
                        acc[cb][d0 + e] = mfma16x16x32<MDT>(
                            u32x4{t[e][h][0], t[e][h][1], t[e][h][0], t[e][h][1]}, pf[cb][h], acc[cb][d0 + e]);
            }
        }
    };

    // Tile i + 1 is in flight while tile i is consumed.
    Cur cq[ST];   // cursors of tiles i ..
    uint64_t gb[GROUPS];
    load_q(ic);
    bool began_here = ic.t == 0;
    group_bases(ic, gb);
    static_assert(ST == 2, "one tile before the loop");
    cq[0] = ic;
    if (n > 0) issue(0, gb, ic.again);
    if (n > 1) {
        advance(ic, t0 + 1);
        group_bases(ic, gb);
    }
    // (one copy of the step: a wave runs it some ten times, and code that is not yet in
    // the instruction cache costs more than the moves)
    uint32_t place = 0, fill = 2 * HALF;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        cq[ST - 1] = ic;
        if (i + ST - 1 < n) {
            issue(fill, gb, ic.again);   // (the place's last reads have returned)
            if (i + ST < n) {
                advance(ic, t0 + i + ST);
                group_bases(ic, gb);
            }
            wait_loads<(ST - 1) * LOADS>();   // tile i is there
        } else {
            wait_loads<0>();
        }
        compute(place, cq[0]);
        if (i + 1 < n) {
            if (cq[0].t == cq[0].nt - 1) {
                flush(cq[0], began_here);
                load_q(cq[1]);   // a new (item, kv head)
                began_here = true;
            }
            cq[0] = cq[1];
        }
        fill = place;
        place ^= 2 * HALF;
    }

    // Waves whose slices end in the same (item, kv head) -- all but the first lie in it
    // wholly -- make one part of theirs, in the place of the first's: a quarter of the
    // parts of a long prefix.
    const Cur& c = cq[0];
    const int key = n > 0 ? (c.own * kMaxRows + c.r) * Hkv + c.g : -1;
    if (lane == 0) {
        s_key[wave] = key;
        s_began[wave] = began_here;
    }
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
        const float l = wave_sum_across_groups(l_run[cb]);
        if (lg == 0) s_ml[wave][cb * 16 + ln] = float2{m_run[cb], l};
    }
    __syncthreads();
    int head = wave, last = wave;   // of the run of waves
    while (head > 0 && uni(s_key[head - 1]) == key) --head;
    while (last + 1 < kWaves && uni(s_key[last + 1]) == key) ++last;
    const int run = key < 0 ? 0 : last - head + 1;
    const bool begins = uni(s_began[head]) != 0;
    constexpr int MOST = ST * 2 * HALF / (DB * 1024);   // column blocks that a ring takes
    constexpr int PASS = MOST < NCB ? MOST : NCB;
    static_assert(PASS >= 1 && NCB % PASS == 0, "outputs pass through the rings");
#pragma unroll
    for (int p0 = 0; p0 < NCB; p0 += PASS) {
        f32x4* const mine = reinterpret_cast<f32x4*>(s_ring[wave]) + lane;
#pragma unroll
        for (int cb = p0; cb < p0 + PASS; ++cb) {
            if (run == 0 || cb >= c.blocks) break;
            float m = -INFINITY, l = 0.0f;
            for (int w = head; w <= last; ++w) m = fmaxf(m, s_ml[w][cb * 16 + ln].x);
            for (int w = head; w <= last; ++w)
                l += s_ml[w][cb * 16 + ln].y * __builtin_amdgcn_exp2f(s_ml[w][cb * 16 + ln].x - m);
            const float weight = __builtin_amdgcn_exp2f(m_run[cb] - m);
#pragma unroll
            for (int db = 0; db < DB; ++db) mine[((cb - p0) * DB + db) * 64] = acc[cb][db] * weight;
            if (wave == head && lg == 0 && seq_of[cb] < c.seqs) *part_ml(c, begins, slice, cb) = float2{m, l};
        }
        __syncthreads();
#pragma unroll
        for (int cb = p0; cb < p0 + PASS; ++cb) {
            if (run == 0 || cb >= c.blocks) break;
            float* const to = part_acc(c, begins, slice - (wave - head), cb);
            const int step = begins ? 16 : 256;
            for (int db = wave - head; db < DB; db += run) {
                f32x4 sum = f32x4{0, 0, 0, 0};
                for (int w = head; w <= last; ++w)
                    sum += reinterpret_cast<const f32x4*>(s_ring[w])[((cb - p0) * DB + db) * 64 + lane];
                if (seq_of[cb] < c.seqs) *reinterpret_cast<f32x4*>(to + db * step) = sum;
            }
        }
        if (p0 + PASS < NCB) __syncthreads();
    }
}

// Joins the parts of a (sequence, kv head) by their log-sum-exp: weights of up
// to kJoin parts at a time in LDS, four outputs a thread, the parts dealt to
// threads that are left over (their sums meet in LDS).  A sequence without tokens
// gets zeros here.
constexpr int kJoin = 64, kJoinThreads = 256;
template <int DT, int D>
__global__ __launch_bounds__(kJoinThreads) void attn_shared_join(FastParams f, int slot_cols) {
    __shared__ float s_w[16][kJoin], s_scale[16], s_inv[16];
    __shared__ f32x4 s_red[kJoinThreads];
    const SharedParams& p = f.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = static_cast<int>(blockIdx.x) / p.kv_heads, g = static_cast<int>(blockIdx.x) - r * p.kv_heads;
    const int G = f.group, Hq = p.num_q_heads;
    const RowPlan w = f.plan[r];
    const int per = f.per[0], total = f.per[1];
    uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + (static_cast<size_t>(f.row0 + r) * Hq + g * G) * D;
    if (w.pre_tiles + w.own_tiles == 0) {
        for (int e = tid; e < G * D; e += kJoinThreads) out[e] = 0;
        return;
    }
    // The parts of a run of tiles from `first` on: of each workgroup whose slices lie in
    // it one, by the place of its first such slice (the first of all in the row of its
    // own), and, where a slice goes on behind the run's end, that slice's.
    struct Parts {
        int first, wgs, n, last;
    };
    auto parts_of = [&](int first, int tiles) {
        Parts q{};
        if (tiles == 0) return q;
        q.first = first / per;
        q.last = (first + tiles - 1) / per;
        const bool on = static_cast<long long>(q.last + 1) * per > first + tiles && first + tiles < total;
        const int whole = q.last - on;   // the last slice that ends in the run
        q.wgs = whole >= q.first ? whole / kWaves - q.first / kWaves + 1 : 0;
        q.n = q.wgs + on;
        return q;
    };
    const Parts pre = parts_of(w.pre_tile + g * f.per[2], w.pre_tiles);
    const Parts own = parts_of(w.own_tile + g * w.own_tiles, w.own_tiles);
    const int parts = pre.n + own.n;
    const int shift = (f.row0 + r - w.first) * G;   // its columns in the item's slices
    // the row of part k's column of head 0: in the first parts' rows, or of a slice
    auto place = [&](int k, bool* first) -> size_t {
        const bool mine = k >= pre.n;
        const Parts& q = mine ? own : pre;
        if (mine) k -= pre.n;
        const int slice = k >= q.wgs ? q.last : k == 0 ? q.first : (q.first / kWaves + k) * kWaves;
        *first = k == 0;
        if (k == 0) return static_cast<size_t>(mine * f.rows + r) * Hq + g * G;
        return static_cast<size_t>(slice) * slot_cols + (mine ? 0 : shift);
    };
    // outputs 4 q .. of heads 0 ..: q % (D / 4) of a row's, of a slice by its registers' order
    auto outputs = [&](int k, int q) {
        bool first;
        const size_t row = place(k, &first);
        if (first) return f.acc + row * D + q * 4;
        const size_t col = row + q / (D / 4);
        const int d = q % (D / 4);
        return f.slice_acc + ((col >> 4) * (D / 16) + (d >> 2)) * 256 + ((d & 3) * 16 + (col & 15)) * 4;
    };
    const int quads = G * D / 4;                       // 16 .. 512
    constexpr int MAXQ = 2;                            // of a thread
    const int threads = min(quads, kJoinThreads);      // on one part
    const int deal = kJoinThreads / threads, lane_q = tid % threads, turn = tid / threads;
    f32x4 acc[MAXQ] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
    float top[4], sum[4];                              // heads wave, wave + 4, ...
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        top[i] = -INFINITY;
        sum[i] = 0.0f;
    }
    for (int k0 = 0; k0 < parts; k0 += kJoin) {
        const int kn = min(kJoin, parts - k0);
        bool first;
        const size_t at = place(k0 + min(lane, kn - 1), &first);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int h = wave + 4 * i;
            if (h >= G) continue;
            const float* ml = (first ? f.ml : f.slice_ml) + (at + h) * 2;
            const float m = lane < kn ? ml[0] : -INFINITY, l = lane < kn ? ml[1] : 0.0f;
            float mx = m;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
            mx = fmaxf(mx, top[i]);
            const float old = top[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[i] - mx);
            const float weight = lane < kn ? __builtin_amdgcn_exp2f(m - mx) : 0.0f;
            float add = weight * l;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) add += __shfl_xor(add, o);
            sum[i] = sum[i] * old + add;
            top[i] = mx;
            s_w[h][lane] = weight;
            if (lane == 0) {
                s_scale[h] = old;
                s_inv[h] = 1.0f / sum[i];
            }
        }
        __syncthreads();
        if (turn < deal) {
#pragma unroll
            for (int i = 0; i < MAXQ; ++i) {
                const int q = lane_q + i * kJoinThreads;
                if (q >= quads) continue;
                const int h = q * 4 / D;
                f32x4 a = acc[i] * s_scale[h];
#pragma unroll 4
                for (int k = turn; k < kn; k += deal) {
                    a += s_w[h][k] * *reinterpret_cast<const f32x4*>(outputs(k0 + k, q));
                }
                acc[i] = a;
            }
        }
        __syncthreads();
    }
    if (deal > 1) {
        s_red[tid] = acc[0];
        __syncthreads();
        if (turn == 0)
            for (int i = 1; i < deal; ++i) acc[0] += s_red[i * threads + lane_q];
    }
    if (turn > 0) return;   // (and where threads are left over that took no part)
#pragma unroll
    for (int i = 0; i < MAXQ; ++i) {
        const int q = lane_q + i * kJoinThreads;
        if (q >= quads) continue;
        const f32x4 a = acc[i] * s_inv[q * 4 / D];
        u32x2 o;
        o[0] = f32_to_elem<DT>(a[0]) | (f32_to_elem<DT>(a[1]) << 16);
        o[1] = f32_to_elem<DT>(a[2]) | (f32_to_elem<DT>(a[3]) << 16);
        *reinterpret_cast<u32x2*>(out + q * 4) = o;
    }
}

// Column blocks of an item: two of 128 elements, or four of 64, are what half of a
// SIMD's registers hold; one where a group has few query rows a kv head (in the mean
// over groups).  One and two, 128 elements, prompts of 1 to 4 thousand: 4 rows 136
// and 140 us, 8 rows 89 and 84 (fp8 64 and 62; two sequences alone 14.1 and 14.8),
// 16 rows 106 and 89; one and four, 64 elements: 8 rows 31.3 and 32.9.
constexpr int kSlices = 2048;   // two workgroups of four waves a CU
int column_blocks(int d, long long rows, int batch) {
    const bool few = rows < 8 || (rows == 8 && (d == 64 || batch < 16));
    return few ? 1 : d == 64 ? 4 : 2;
}

// Where things lie in the scratch of a launch of `rows` sequences.
struct Layout {
    size_t per, plan, ml, slice_ml, acc, slice_acc, bytes;
};
Layout layout_of(int rows, int hq, int d, int ncb) {
    Layout l{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~size_t(255);
        return here;
    };
    const size_t firsts = size_t(2) * rows * hq, later = static_cast<size_t>(kSlices) * 16 * ncb;
    l.per = take(3 * sizeof(int));
    l.plan = take(static_cast<size_t>(rows) * sizeof(RowPlan));
    l.ml = take(firsts * 8);
    l.slice_ml = take(later * 8);
    l.acc = take(firsts * d * 4);
    l.slice_acc = take(later * d * 4);
    l.bytes = at;
    return l;
}

bool fast_shape(int dtype, uint32_t hq, uint32_t hkv, uint32_t d, uint32_t bs) {
    int flag = 0;
    return dtype != kDtF32 && hq % hkv == 0 && hq / hkv <= 16 && bs % 8 == 0 &&
           (d == 128 || (d == 64 && dtype != kDtFP8)) && !dev::tunable(dev::Tun::kAttnGeneric, &flag);
}

template <int DT, int D, int NCB>
bool launch_fast(const SharedParams& p, uint64_t scratch, hipStream_t s, std::string* err) {
    FastParams f{};
    f.p = p;
    f.group = p.num_q_heads / p.kv_heads;
    f.seqs = 16 * NCB / f.group;
    f.scale_log2 = p.scale * 1.4426950408889634f;
    f.slices = kSlices;
    const long long cap = static_cast<long long>(p.mbps) * p.block_size;
    for (int row0 = 0; row0 < p.batch; row0 += kMaxRows) {
        f.row0 = row0;
        f.rows = std::min(kMaxRows, p.batch - row0);
        if (2LL * f.rows * p.kv_heads * ((cap + 15) / 16) > (1LL << 30)) {
            *err = "batch x context too large";
            return false;
        }
        const Layout l = layout_of(f.rows, p.num_q_heads, D, NCB);
        auto at = [&](size_t o) { return reinterpret_cast<float*>(scratch + o); };
        f.per = reinterpret_cast<int*>(scratch + l.per);
        f.plan = reinterpret_cast<RowPlan*>(scratch + l.plan);
        f.ml = at(l.ml);
        f.slice_ml = at(l.slice_ml);
        f.acc = at(l.acc);
        f.slice_acc = at(l.slice_acc);
        // no more workgroups than the tables hold tiles for
        const long long most = 2LL * f.rows * p.kv_heads * ((cap + 15) / 16);
        const unsigned wgs = static_cast<unsigned>(std::min<long long>(f.slices, most) + kWaves - 1) / kWaves;
        auto run = [&](auto bs) {
            hipLaunchKernelGGL((attn_shared_stream<DT, D, decltype(bs)::value, NCB>), dim3(wgs),
                               dim3(64 * kWaves), 0, s, f, p.block_tables, p.offsets_f16, p.k_base, p.v_base);
        };
        if (p.block_size == 16) run(std::integral_constant<int, 16>{});
        else run(std::integral_constant<int, 0>{});
        KCMM_HIP_CHECK(hipGetLastError(), err);
        hipLaunchKernelGGL((attn_shared_join<DT == kDtFP8 ? kDtBF16 : DT, D>),
                           dim3(static_cast<unsigned>(f.rows * p.kv_heads)), dim3(kJoinThreads), 0, s, f, 16 * NCB);
        KCMM_HIP_CHECK(hipGetLastError(), err);
    }
    return true;
}

template <int DT, int D>
bool launch_columns(const SharedParams& p, uint64_t scratch, hipStream_t s, std::string* err) {
    const long long rows = static_cast<long long>(p.batch) * (p.num_q_heads / p.kv_heads) / p.groups;
    return column_blocks(D, rows, p.batch) == 1 ? launch_fast<DT, D, 1>(p, scratch, s, err)
                                       : launch_fast<DT, D, D == 64 ? 4 : 2>(p, scratch, s, err);
}

// Enough for either number of column blocks.
uint64_t fast_scratch(uint32_t batch, uint32_t num_q_heads, uint32_t head_dim) {
    const int rows = static_cast<int>(std::min<uint32_t>(batch, kMaxRows));
    const int hq = static_cast<int>(num_q_heads), d = static_cast<int>(head_dim);
    return std::max(layout_of(rows, hq, d, 1).bytes, layout_of(rows, hq, d, column_blocks(d, INT_MAX, INT_MAX)).bytes);
}

}  // namespace

namespace dev {

uint64_t attn_shared_scratch_bytes(int32_t dtype, uint32_t batch, uint32_t num_q_heads, uint32_t kv_heads,
                                   uint32_t head_dim, uint32_t block_size, uint32_t) {
    if (!fast_shape(dtype, num_q_heads, kv_heads, head_dim, block_size)) return 256;
    return fast_scratch(batch, num_q_heads, head_dim);
}

bool attn_shared(const AttnSharedArgs& a, std::string* err) {
    SharedParams p{};
    p.q = reinterpret_cast<const uint8_t*>(a.q);
    p.out = reinterpret_cast<uint8_t*>(a.out);
    p.k_base = reinterpret_cast<const uint8_t*>(a.k_base);
    p.v_base = reinterpret_cast<const uint8_t*>(a.v_base);
    p.block_tables = reinterpret_cast<const int32_t*>(a.block_tables);
    p.seq_lens = reinterpret_cast<const int32_t*>(a.seq_lens);
    p.shared_lens = reinterpret_cast<const int32_t*>(a.shared_lens);
    p.group_starts = reinterpret_cast<const int32_t*>(a.group_starts);
    p.offsets_f16 = reinterpret_cast<const uint64_t*>(a.offsets_f16);
    p.batch = static_cast<int>(a.batch);
    p.groups = static_cast<int>(a.num_groups);
    p.num_q_heads = static_cast<int>(a.num_q_heads);
    p.kv_heads = static_cast<int>(a.kv_heads);
    p.head_dim = static_cast<int>(a.head_dim);
    p.block_size = static_cast<int>(a.block_size);
    p.mbps = static_cast<int>(a.mbps);
    p.row_bytes = static_cast<int>(a.row_bytes);
    p.data_bytes = static_cast<int>(a.data_bytes);
    p.scale = a.scale;
    hipStream_t s = reinterpret_cast<hipStream_t>(a.stream);
    if (fast_shape(a.dtype, a.num_q_heads, a.kv_heads, a.head_dim, a.block_size)) {
        // (again: the caller's check may have been of another choice of kernels)
        if (a.scratch_bytes < fast_scratch(a.batch, a.num_q_heads, a.head_dim)) {
            *err = "scratch is too small";
            return false;
        }
        if (a.dtype == kDtFP8) return launch_columns<kDtFP8, 128>(p, a.scratch, s, err);
        if (a.dtype == kDtF16)
            return a.head_dim == 64 ? launch_columns<kDtF16, 64>(p, a.scratch, s, err)
                                    : launch_columns<kDtF16, 128>(p, a.scratch, s, err);
        return a.head_dim == 64 ? launch_columns<kDtBF16, 64>(p, a.scratch, s, err)
                                : launch_columns<kDtBF16, 128>(p, a.scratch, s, err);
    }
    switch (a.dtype) {
        case kDtF16: launch_generic<kDtF16>(p, s); break;
        case kDtBF16: launch_generic<kDtBF16>(p, s); break;
        case kDtF32: launch_generic<kDtF32>(p, s); break;
        default: launch_generic<kDtFP8>(p, s); break;
    }
    KCMM_HIP_CHECK(hipGetLastError(), err);
    return true;
}

}  // namespace dev
}  // namespace kcmm
