// Paged decode attention of groups of sequences that share a prefix (gfx950).
//
//   out[b][h] = sum_t softmax_t(scale q[b][h].K[t]) V[t],  t < L_b,
// the whole blocks among the first min(shared_lens[b], L_b) tokens of sequence b
// (s_b tokens) being those of the first sequence of its group, through whose
// table they are read; the rest is read through b's own table.  L_b <= 0 writes
// zeros.  Sums, maxima and outputs are fp32 up to the store.
//
// Bound by HBM: a page that a group shares is read once for up to 64 / G of its
// sequences (G query heads a kv head), instead of once for each.
//  * An item is a run of sequences of one group with the tokens that they have in
//    common, or one sequence with the tokens behind those.  16 NCB columns of the
//    matrix products are (sequence of the item, query head) pairs, so a K/V byte
//    in registers serves up to 64 query rows, as one of a single sequence serves
//    G.  No column of an item is masked: a sequence that shares less than half of
//    what the others do is left to read its tokens by itself.
//  * The work is the list of 32-token tiles of all (item, kv head), common tokens
//    first; every wave takes an equal, contiguous slice of it and streams its
//    pages through registers, the next tile's loads in flight.  Each workgroup
//    works out items and slices for itself, from lengths and group starts, in LDS
//    (a kernel in front would cost more than that).
//  * S^T = K Q^T and O^T += V^T P^T on 16x16x32 matrix instructions, softmax with a
//    running maximum in the log2 domain; V is turned by the transposing LDS read,
//    through LDS of the wave's own (no barrier in the loop).
//  * Parts of a (sequence, head) -- slices of the common tokens, slices of the rest
//    -- are joined by their log-sum-exp in a second kernel.
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
    float m = -INFINITY, s = 0.0f;
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
            const float corr = m == -INFINITY ? 0.0f : kexp<DT>(m - top);
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
    const float f = m == -INFINITY ? 0.0f : kexp<DT>(m - M);
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
        float top = -INFINITY, S = 0.0f, o = 0.0f;
        for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, s_m[w]);
        for (int w = 0; w < kThreads / 64; ++w) {
            const float e = s_m[w] == -INFINITY ? 0.0f : kexp<DT>(s_m[w] - top);
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

constexpr int kWaves = 4;          // of a workgroup
constexpr int kMaxRows = 512;      // sequences of a launch
constexpr int kRowsPerThread = kMaxRows / (64 * kWaves);

// What the joining kernel has to know of a sequence: where its parts are.
struct RowPlan {
    int pre_tile, pre_tiles;   // first tile of the item's common tokens (kv head 0), tiles a kv head; 0: none
    int first;                 // first sequence of the item
    int own_tile, own_tiles;   // the same of the tokens behind them
};

struct FastParams {
    SharedParams p;
    int row0, rows;            // sequences of this launch
    int group, seqs;           // query heads a kv head; sequences of an item
    int slices, least;         // waves; least tiles of one
    int* per;                  // tiles of a slice, for the joining kernel
    RowPlan* plan;
    // first parts of (sequence, head): of the common tokens, then of the rest;
    // later parts by slice, a row a column
    float *ml, *acc, *slice_ml, *slice_acc;
    float scale_log2;
};

__device__ __forceinline__ int tiles_of(int tokens) { return (tokens + 31) >> 5; }

// Exclusive sums over kMaxRows values, kRowsPerThread consecutive ones a thread;
// *all: their sum.  s_wave: kWaves ints of LDS.
__device__ __forceinline__ void block_sums(const int (&v)[kRowsPerThread], int (&at)[kRowsPerThread], int* all,
                                           int* s_wave) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = 0;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        at[i] = sum;
        sum += v[i];
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    int before = incl - sum;
    *all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += s_wave[w];
        *all += s_wave[w];
    }
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) at[i] += before;
    __syncthreads();
}

// The items of this launch, in LDS, by sequence (relative to row0).
struct Items {
    int len[kMaxRows];      // tokens, clamped to what the table holds
    int shared[kMaxRows];   // tokens in shared blocks
    int lead[kMaxRows];     // whose table these are read through (of the whole batch)
    int common[kMaxRows];   // tokens that the item of the sequence takes in common; 0: none
    int count[kMaxRows];    // sequences of the item that begins here, 0: none does
    int most[kMaxRows];     // its common tokens
    int pre[kMaxRows];      // tiles of the items before this sequence, of one kv head
    int own[kMaxRows];      // the same of the sequences' own tokens
    int pre_all, own_all;
    int wave[kWaves];
    int carry;
};

__device__ __forceinline__ void find_items(const FastParams& f, Items& it) {
    const SharedParams& p = f.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr int N = kRowsPerThread;
    const int cap = p.mbps * p.block_size, r0 = tid * N;
    int len[N], want[N], lead[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + i;
        len[i] = want[i] = 0;
        if (r < f.rows) {
            len[i] = max(0, min(p.seq_lens[f.row0 + r], cap));
            want[i] = p.shared_lens[f.row0 + r];
        }
        it.lead[r] = -1;
        it.common[r] = it.count[r] = 0;
    }
    if (tid == 0) it.carry = -1;
    __syncthreads();
    const int end = p.group_starts[p.groups];   // sequences from here on lie in no group
    for (int g = tid; g < p.groups; g += 64 * kWaves) {
        const int start = p.group_starts[g];
        if (start < 0 || start >= p.batch) continue;
        if (start >= f.row0 && start < f.row0 + f.rows) atomicMax(&it.lead[start - f.row0], start);
        else if (start < f.row0) atomicMax(&it.carry, start);
    }
    __syncthreads();
    // the last group start not behind a sequence
    int top = -1;
#pragma unroll
    for (int i = 0; i < N; ++i) lead[i] = top = max(top, it.lead[r0 + i]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(top, o);
        if (lane >= o) top = max(top, y);
    }
    if (lane == 63) it.wave[wave] = top;
    int before = __shfl_up(top, 1);
    if (lane == 0) before = -1;
    __syncthreads();
    before = max(before, it.carry);
    for (int w = 0; w < wave; ++w) before = max(before, it.wave[w]);
    unsigned begins = 0;   // bit i: an item begins at r0 + i
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + i, b = f.row0 + r;
        lead[i] = max(lead[i], before);
        const bool in = r < f.rows && lead[i] >= 0 && b < end;
        it.len[r] = len[i];
        it.shared[r] = in ? whole_blocks(min(want[i], len[i]), p.block_size) : 0;
        it.lead[r] = in ? lead[i] : -1;
        if (in && (b - max(lead[i], f.row0)) % f.seqs == 0) begins |= 1u << i;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
        if (!(begins >> i & 1)) continue;
        const int r = r0 + i, mine = it.lead[r];
        const int last = min(r + f.seqs, f.rows);
        int most = 0, n = 0;
        for (; r + n < last && it.lead[r + n] == mine; ++n) most = max(most, it.shared[r + n]);
        int common = most, part = 0;
        for (int j = 0; j < n; ++j) {
            const int s = it.shared[r + j];
            if (2 * static_cast<long long>(s) < most) continue;
            common = min(common, s);
            ++part;
        }
        if (common <= 0 || part < 2) continue;   // nothing to gain: each reads its own
        it.count[r] = n;
        it.most[r] = common;
        for (int j = 0; j < n; ++j)
            if (it.shared[r + j] >= common) it.common[r + j] = common;
    }
    __syncthreads();
    int pre[N], own[N], at[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + i;
        pre[i] = it.count[r] > 0 ? tiles_of(it.most[r]) : 0;   // (the first sequence need not take part)
        own[i] = tiles_of(it.len[r] - it.common[r]);
    }
    int all;
    block_sums(pre, at, &all, it.wave);
#pragma unroll
    for (int i = 0; i < N; ++i) it.pre[r0 + i] = at[i];
    if (tid == 0) it.pre_all = all;
    block_sums(own, at, &all, it.wave);
#pragma unroll
    for (int i = 0; i < N; ++i) it.own[r0 + i] = at[i];
    if (tid == 0) it.own_all = all;
    __syncthreads();
}

// Tiles of a slice: equal parts of all, but none so short that joining the parts
// costs more than the shorter slices save.
__device__ __forceinline__ int slice_tiles(int total, const FastParams& f) {
    return max((total + f.slices - 1) / f.slices, f.least);
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
template <int O0, int O1>
__device__ __forceinline__ void lds_read(u32x4 (&x)[2][4], const uint32_t (&a)[4]) {
    asm volatile("ds_read_b128 %0, %8 offset:%12\n\tds_read_b128 %1, %9 offset:%12\n\t"
                 "ds_read_b128 %2, %10 offset:%12\n\tds_read_b128 %3, %11 offset:%12\n\t"
                 "ds_read_b128 %4, %8 offset:%13\n\tds_read_b128 %5, %9 offset:%13\n\t"
                 "ds_read_b128 %6, %10 offset:%13\n\tds_read_b128 %7, %11 offset:%13\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[0][2]), "=&v"(x[0][3]), "=&v"(x[1][0]),
                   "=&v"(x[1][1]), "=&v"(x[1][2]), "=&v"(x[1][3])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(O0), "i"(O1) : "memory");
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
template <int O>
__device__ __forceinline__ void lds_write(uint32_t a, u32x4 x) {
    asm volatile("ds_write_b128 %0, %1 offset:%2" :: "v"(a), "v"(x), "i"(O) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)p));
}

template <int DT, int D, int BS, int NCB>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(NCB == 1 ? 2 : 1)))
void attn_shared_stream(FastParams f, const int32_t* __restrict__ bt, const uint64_t* __restrict__ offs,
                        const uint8_t* __restrict__ kreg, const uint8_t* __restrict__ vreg,
                        const uint8_t* __restrict__ idle) {
    constexpr bool F8 = DT == kDtFP8;
    constexpr int MDT = F8 ? kDtBF16 : DT;     // matrix, q and out element type
    constexpr int EB = F8 ? 1 : 2;
    constexpr int KC = D / 32, DB = D / 16;
    constexpr int ROWB = D * EB;               // bytes of a token's head row
    constexpr int HALF = 32 * ROWB;            // of a tile's K, and of its V
    constexpr int LOADS = 2 * HALF / 1024;     // of a tile
    constexpr int ST = ROWB == 256 ? 2 : F8 ? 3 : 4;   // tiles of the ring
    constexpr int VROW = 2 * D + 32;           // bytes of a padded V row (fp8)
    static_assert(!F8 || D == 128, "fp8 pages take this path at head_dim 128");
    __shared__ Items it;
    __shared__ __attribute__((aligned(1024))) uint8_t s_ring[kWaves][ST * 2 * HALF];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[F8 ? kWaves : 1][F8 ? 32 * VROW : 16];
    const SharedParams& p = f.p;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int ln = lane & 15, lg = lane >> 4;
    const int bs = BS > 0 ? BS : p.block_size;
    const int Hkv = p.kv_heads, Hq = p.num_q_heads, G = f.group;
    auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };

    find_items(f, it);
    const int pre_end = uni(it.pre_all) * Hkv, total = pre_end + uni(it.own_all) * Hkv;
    const int per = slice_tiles(total, f);
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) *f.per = per;
        int first = -1;
        for (int r = threadIdx.x; r < f.rows; r += 64 * kWaves) {
            RowPlan w{};
            w.own_tile = pre_end + it.own[r] * Hkv;
            w.own_tiles = tiles_of(it.len[r] - it.common[r]);
            if (it.common[r] > 0) {
                first = r;   // the item that r lies in begins at most seqs - 1 before
                while (it.count[first] == 0) --first;
                w.first = f.row0 + first;
                w.pre_tile = it.pre[first] * Hkv;
                w.pre_tiles = tiles_of(it.common[r]);
            }
            f.plan[r] = w;
        }
    }
    const int slice = static_cast<int>(blockIdx.x) * kWaves + wave;
    const long long t0l = static_cast<long long>(slice) * per;
    if (t0l >= total) return;
    const int t0 = static_cast<int>(t0l), n = min(per, total - t0);

    // Cursor over the tile list: tokens begin + 32 t .. of (item, kv head); all of it
    // wave-uniform, so that the tables are read by scalar loads
    struct Cur {
        int r, own, g, t, nt, begin, end, shared, lead, cols;
        float ks[F8 ? 4 : 1], vs[F8 ? 4 : 1];   // fp8: page scales of the 8-token groups
    };
    auto locate = [&](int tile) __attribute__((always_inline)) {
        Cur c;
        c.own = tile >= pre_end;
        const int* sums = c.own ? it.own : it.pre;
        const int rel = c.own ? tile - pre_end : tile, x = rel / Hkv;
        int lo = 0, hi = f.rows;   // the last sequence with sums[r] <= x: it has tiles
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (uni(sums[mid]) <= x) lo = mid;
            else hi = mid;
        }
        c.r = lo;
        const int n_seqs = c.own ? 1 : uni(it.count[lo]);
        const int common = uni(c.own ? it.common[lo] : it.most[lo]);
        c.cols = n_seqs * G;
        c.begin = c.own ? common : 0;
        c.end = c.own ? uni(it.len[lo]) : common;
        c.shared = c.own ? uni(it.shared[lo]) : common;
        c.lead = max(uni(it.lead[lo]), 0);
        c.nt = max(tiles_of(c.end - c.begin), 1);
        const int rem = rel - uni(sums[lo]) * Hkv;
        c.g = rem / c.nt;
        c.t = rem - c.g * c.nt;
        return c;
    };
    Cur ic = locate(t0);
    // (tile: the cursor's new place in the list)
    auto advance = [&](Cur& c, int tile) __attribute__((always_inline)) {
        if (++c.t < c.nt) return;
        c.t = 0;
        if (++c.g == Hkv) c = locate(tile);
    };
    // Page-relative address of each 8-token group of a tile; groups past the end
    // re-read the last one (masked).  fp8: also the groups' page scales.
    auto group_bases = [&](Cur& c, uint64_t* gb) __attribute__((always_inline)) {
        const int last8 = (c.end - 1) & ~7;
        const int32_t* mine = bt + static_cast<size_t>(f.row0 + c.r) * p.mbps;
        const int32_t* theirs = bt + static_cast<size_t>(c.lead) * p.mbps;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int tok = min(c.begin + c.t * 32 + q * 8, last8);
            const int lb = tok / bs;
            const uint64_t page = offs[(tok < c.shared ? theirs : mine)[lb]] * 2ull;
            gb[q] = page + static_cast<uint32_t>((tok - lb * bs) * p.row_bytes + c.g * D * EB);
            if constexpr (F8) {
                const uint64_t sc = page + static_cast<uint32_t>(p.data_bytes + c.g * 4);
                c.ks[q] = *reinterpret_cast<const float*>(kreg + sc);
                c.vs[q] = *reinterpret_cast<const float*>(vreg + sc);
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
    auto issue = [&](int place, bool real, const uint64_t* gb) __attribute__((always_inline)) {
        const uint8_t* kb = real ? kreg : idle;
        const uint8_t* vb = real ? vreg : idle;
        uint8_t* const to = ring + place * 2 * HALF;
#pragma unroll
        for (int i = 0; i < 32 / ROWS; ++i) {
            const uint64_t g = real ? gb[i * ROWS / 8] : 0;
            load_lds16_nt(kb + g + src[i % STEP], to + i * 1024);
            load_lds16_nt(vb + g + src[i % STEP], to + HALF + i * 1024);
        }
    };
    // Column c of an item: head c % G of the kv head's, of its sequence c / G.
    // Columns past the last repeat it; they are computed and never stored.
    u32x4 qf[NCB][KC];
    auto load_q = [&](const Cur& c) __attribute__((always_inline)) {
        const int cols = c.cols;
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            const int col = min(cb * 16 + ln, cols - 1), s = col / G;
            const uint8_t* qrow =
                p.q + (static_cast<size_t>(f.row0 + c.r + s) * Hq + c.g * G + (col - s * G)) * D * 2;
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
            m_run[cb] = -3.402823466e38f;   // (finite: a first tile of scores -inf leaves 0, no NaN)
            l_run[cb] = 0.0f;
#pragma unroll
            for (int i = 0; i < DB; ++i) acc[cb][i] = f32x4{0, 0, 0, 0};
        }
    };
    clear();

    auto flush = [&](const Cur& c, bool began_here) __attribute__((always_inline)) {
        const bool complete = began_here && c.t == c.nt - 1;
        const int cols = c.cols;
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            const float l = wave_sum_across_groups(l_run[cb]);
            const int col = cb * 16 + ln;
            if (col >= cols) continue;
            const int s = col / G, row = c.r + s, h = c.g * G + (col - s * G);
            if (complete && c.own && c.begin == 0) {
                const float inv = 1.0f / l;
                uint16_t* o = reinterpret_cast<uint16_t*>(p.out) +
                              (static_cast<size_t>(f.row0 + row) * Hq + h) * D + 4 * lg;
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    u32x2 w;
                    w[0] = f32_to_elem<MDT>(acc[cb][db][0] * inv) | (f32_to_elem<MDT>(acc[cb][db][1] * inv) << 16);
                    w[1] = f32_to_elem<MDT>(acc[cb][db][2] * inv) | (f32_to_elem<MDT>(acc[cb][db][3] * inv) << 16);
                    *reinterpret_cast<u32x2*>(o + 16 * db) = w;
                }
                continue;
            }
            // the part where a (sequence, head) begins has a row of its own, later
            // ones take the slice's
            const size_t at = began_here ? static_cast<size_t>(c.own * f.rows + row) * Hq + h
                                         : static_cast<size_t>(slice) * (16 * NCB) + col;
            float* pa = (began_here ? f.acc : f.slice_acc) + at * D + 4 * lg;
            float* ml = (began_here ? f.ml : f.slice_ml) + at * 2;
#pragma unroll
            for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(pa + 16 * db) = acc[cb][db];
            if (lg == 0) {
                ml[0] = m_run[cb];
                ml[1] = l;
            }
        }
        clear();
    };

    // this lane's places in a tile: pieces of K's operand rows, of V's transposed ones,
    // and where it writes V's (fp8: as bf16, in padded rows)
    constexpr int NP = F8 ? KC / 2 : KC;
    const uint32_t at0 = lds_address(ring);
    uint32_t k_at[NP], v_at[DB];
#pragma unroll
    for (int i = 0; i < NP; ++i) k_at[i] = at0 + turned(ln, 4 * i + lg);
    const uint32_t sv_at = lds_address(s_v[F8 ? wave : 0]);
#pragma unroll
    for (int db = 0; db < DB; ++db) {
        const int row = 4 * lg + (ln >> 2);
        v_at[db] = F8 ? sv_at + row * VROW + db * 32 + (ln & 3) * 8
                      : at0 + turned(row, 2 * db + ((ln & 3) >> 1)) + (ln & 1) * 8;
    }
    auto compute = [&](auto where, const Cur& c) __attribute__((always_inline)) {
        constexpr int TK = decltype(where)::value * 2 * HALF, TV = TK + HALF;
        const int tbase = c.begin + c.t * 32;
        // rows past the end may hold anything and become zeros
        if (tbase + 32 > c.end)
            for (int row = c.end - tbase + lane / PIECES; row < 32; row += ROWS)
                lds_write<TV>(at0 + row * ROWB + lane % PIECES * 16, u32x4{0, 0, 0, 0});
        if constexpr (F8) {
            // V as bf16 (exactly: the pages' scales go to P)
            u32x4 x[2][NP];
            lds_read<TV, TV + 16 * ROWB>(x, k_at);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t at = sv_at + (16 * h + ln) * VROW + (4 * e + lg) * 32;
                    lds_write<0>(at, fp8x8_to_bf16(x[h][e][0], x[h][e][1]));
                    lds_write<16>(at, fp8x8_to_bf16(x[h][e][2], x[h][e][3]));
                }
        }
        f32x4 s[NCB][2];
        {
            u32x4 x[2][NP];
            lds_read<TK, TK + 16 * ROWB>(x, k_at);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int cb = 0; cb < NCB; ++cb) s[cb][h] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    u32x4 a = x[h][F8 ? kc >> 1 : kc];
                    if constexpr (F8) a = (kc & 1) ? fp8x8_to_bf16(a[2], a[3]) : fp8x8_to_bf16(a[0], a[1]);
#pragma unroll
                    for (int cb = 0; cb < NCB; ++cb) s[cb][h] = mfma16x16x32<MDT>(a, qf[cb][kc], s[cb][h]);
                }
            }
        }
        u32x4 pf[NCB];
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) {
            float v[8];
            float mt = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float sc = f.scale_log2;
                if constexpr (F8) sc *= lg < 2 ? c.ks[2 * h] : c.ks[2 * h + 1];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float x = tbase + h * 16 + lg * 4 + r < c.end ? s[cb][h][r] * sc : -INFINITY;
                    v[h * 4 + r] = x;
                    mt = fmaxf(mt, x);
                }
            }
            const float m_new = fmaxf(m_run[cb], wave_max_across_groups(mt));
            const float corr = __builtin_amdgcn_exp2f(m_run[cb] - m_new);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = __builtin_amdgcn_exp2f(v[i] - m_new);
                sum += v[i];
            }
            l_run[cb] = l_run[cb] * corr + sum;
            m_run[cb] = m_new;
            if (__any(corr != 1.0f)) {
#pragma unroll
                for (int i = 0; i < DB; ++i) acc[cb][i] *= corr;
            }
            if constexpr (F8) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float vs = lg < 2 ? c.vs[2 * h] : c.vs[2 * h + 1];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[h * 4 + r] *= vs;
                }
            }
            // slots (lg, i) of the P^T operand: token i < 4 ? 4 lg + i : 16 + 4 lg + i - 4
#pragma unroll
            for (int i = 0; i < 4; ++i)
                pf[cb][i] = f32_to_elem<MDT>(v[2 * i]) | (f32_to_elem<MDT>(v[2 * i + 1]) << 16);
        }
#pragma unroll
        for (int d0 = 0; d0 < DB; d0 += 4) {
            // lane (ln, lg): V[4 lg .. +3][16 db + ln], and of the second half
            u32x2 x[4][2];
            const uint32_t at[4] = {v_at[d0], v_at[d0 + 1], v_at[d0 + 2], v_at[d0 + 3]};
            lds_read_turned<F8 ? 0 : TV, F8 ? 16 * VROW : TV + 16 * ROWB>(x, at);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u32x4 vt{x[e][0][0], x[e][0][1], x[e][1][0], x[e][1][1]};
#pragma unroll
                for (int cb = 0; cb < NCB; ++cb)
                    acc[cb][d0 + e] = mfma16x16x32<MDT>(vt, pf[cb], acc[cb][d0 + e]);
            }
        }
    };

    // Tiles i + 1 .. i + ST - 1 are in flight while tile i is consumed, the addresses of
    // tile i + ST are being fetched.  Past the slice's end loads of `idle` (in L2)
    // keep the count of loads in flight the same.
    Cur cq[ST];
    uint64_t gb[4];
    load_q(ic);
    bool began_here = ic.t == 0;
    group_bases(ic, gb);
#pragma unroll
    for (int k = 0; k < ST - 1; ++k) {
        cq[k] = ic;
        issue(k, k < n, gb);
        if (k + 1 < n) {
            advance(ic, t0 + k + 1);
            group_bases(ic, gb);
        }
    }
    auto step = [&](auto phase, int i) __attribute__((always_inline)) {
        constexpr int j = decltype(phase)::value, jn = (j + ST - 1) % ST;
        cq[jn] = ic;
        issue(jn, i + ST - 1 < n, gb);   // (the place's last reads have returned)
        if (i + ST < n) {
            advance(ic, t0 + i + ST);
            group_bases(ic, gb);
        }
        wait_vm_lgkm0<(ST - 1) * LOADS>();   // tile i is there
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (i < n) {
            compute(phase, cq[j]);
            if (i == n - 1 || cq[j].t == cq[j].nt - 1) flush(cq[j], began_here);
            if (i + 1 < n && cq[(j + 1) % ST].t == 0) {
                load_q(cq[(j + 1) % ST]);
                began_here = true;
            }
        }
    };
    for (int i = 0; i < n; i += ST) {
        step(std::integral_constant<int, 0>{}, i);
        step(std::integral_constant<int, 1>{}, i + 1);
        if constexpr (ST > 2) step(std::integral_constant<int, 2>{}, i + 2);
        if constexpr (ST > 3) step(std::integral_constant<int, 3>{}, i + 3);
    }
    // no load may land in LDS that the next workgroup has
    wait_vm_lgkm0<0>();
}

// Joins the parts of a (sequence, kv head) by their log-sum-exp: weights of up
// to kJoin parts at a time in LDS, four outputs a thread, the parts dealt to
// threads that are left over (their sums meet in LDS).  A sequence of one part
// was stored by the streaming kernel; one without tokens gets zeros here.
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
    const int per = *f.per;
    uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + (static_cast<size_t>(f.row0 + r) * Hq + g * G) * D;
    if (w.pre_tiles + w.own_tiles == 0) {
        for (int e = tid; e < G * D; e += kJoinThreads) out[e] = 0;
        return;
    }
    // first slice and slices of the two kinds of parts
    const int pre0 = w.pre_tile + g * w.pre_tiles, own0 = w.own_tile + g * w.own_tiles;
    const int pre_at = pre0 / per, own_at = own0 / per;
    const int pre_n = w.pre_tiles == 0 ? 0 : (pre0 + w.pre_tiles - 1) / per - pre_at + 1;
    const int own_n = w.own_tiles == 0 ? 0 : (own0 + w.own_tiles - 1) / per - own_at + 1;
    if (pre_n == 0 && own_n == 1) return;
    const int parts = pre_n + own_n;
    const int shift = (f.row0 + r - w.first) * G;   // its columns in the item's slices
    // the row of part k's column of head 0: in the first parts' rows, or a slice's
    auto place = [&](int k, bool* first) -> size_t {
        const bool own = k >= pre_n;
        if (own) k -= pre_n;
        *first = k == 0;
        if (k == 0) return static_cast<size_t>(own * f.rows + r) * Hq + g * G;
        return static_cast<size_t>((own ? own_at : pre_at) + k) * slot_cols + (own ? 0 : shift);
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
                    bool one;
                    const size_t row = place(k0 + k, &one);
                    a += s_w[h][k] * *reinterpret_cast<const f32x4*>((one ? f.acc : f.slice_acc) + row * D + q * 4);
                }
                acc[i] = a;
            }
        }
        __syncthreads();
    }
    if (deal > 1) {
        s_red[tid] = acc[0];
        __syncthreads();
        if (turn > 0) return;
        for (int i = 1; i < deal; ++i) acc[0] += s_red[i * threads + lane_q];
    }
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

// Column blocks of an item: as many as a group's query rows fill, up to 64 columns.
int column_blocks(long long rows_of_a_group) { return rows_of_a_group <= 16 ? 1 : rows_of_a_group <= 32 ? 2 : 4; }
int slices_of(int dtype, int ncb) { return dtype == kDtFP8 && ncb == 1 ? 2048 : 1024; }

// Where things lie in the scratch of a launch of `rows` sequences.
struct Layout {
    size_t idle, per, plan, ml, slice_ml, acc, slice_acc, bytes;
};
Layout layout_of(int dtype, int rows, int hq, int d, int row_bytes, int ncb) {
    Layout l{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~size_t(255);
        return here;
    };
    const size_t firsts = size_t(2) * rows * hq, later = static_cast<size_t>(slices_of(dtype, ncb)) * 16 * ncb;
    l.idle = take(static_cast<size_t>(8) * row_bytes + 1024);   // must cover one tile's lane addresses
    l.per = take(sizeof(int));
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
    f.slices = slices_of(DT, NCB);
    f.least = 1;
    const long long cap = static_cast<long long>(p.mbps) * p.block_size;
    for (int row0 = 0; row0 < p.batch; row0 += kMaxRows) {
        f.row0 = row0;
        f.rows = std::min(kMaxRows, p.batch - row0);
        if (2LL * f.rows * p.kv_heads * ((cap + 31) / 32) > (1LL << 30)) {
            *err = "batch x context too large";
            return false;
        }
        const Layout l = layout_of(DT, f.rows, p.num_q_heads, D, p.row_bytes, NCB);
        auto at = [&](size_t o) { return reinterpret_cast<float*>(scratch + o); };
        f.per = reinterpret_cast<int*>(scratch + l.per);
        f.plan = reinterpret_cast<RowPlan*>(scratch + l.plan);
        f.ml = at(l.ml);
        f.slice_ml = at(l.slice_ml);
        f.acc = at(l.acc);
        f.slice_acc = at(l.slice_acc);
        const auto* idle = reinterpret_cast<const uint8_t*>(scratch + l.idle);
        // no more workgroups than the tables hold tiles for
        const long long most = 2LL * f.rows * p.kv_heads * ((cap + 31) / 32);
        const unsigned wgs = static_cast<unsigned>(std::min<long long>(f.slices, most) + kWaves - 1) / kWaves;
        auto run = [&](auto bs) {
            hipLaunchKernelGGL((attn_shared_stream<DT, D, decltype(bs)::value, NCB>), dim3(wgs),
                               dim3(64 * kWaves), 0, s, f, p.block_tables, p.offsets_f16, p.k_base, p.v_base, idle);
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
    switch (column_blocks(rows)) {
        case 1: return launch_fast<DT, D, 1>(p, scratch, s, err);
        case 2: return launch_fast<DT, D, 2>(p, scratch, s, err);
        default: return launch_fast<DT, D, 4>(p, scratch, s, err);
    }
}

}  // namespace

namespace dev {

uint64_t attn_shared_scratch_bytes(int32_t dtype, uint32_t batch, uint32_t num_q_heads, uint32_t kv_heads,
                                   uint32_t head_dim, uint32_t block_size, uint32_t) {
    if (!fast_shape(dtype, num_q_heads, kv_heads, head_dim, block_size)) return 256;
    const int rows = static_cast<int>(std::min<uint32_t>(batch, kMaxRows));
    const int row_bytes = static_cast<int>(kv_heads * head_dim * (dtype == kDtFP8 ? 1 : 2));
    size_t most = 0;
    for (int ncb : {1, 2, 4})
        most = std::max(most, layout_of(dtype, rows, static_cast<int>(num_q_heads), static_cast<int>(head_dim),
                                        row_bytes, ncb).bytes);
    return most;
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
