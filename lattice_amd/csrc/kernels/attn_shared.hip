// Paged decode attention of groups of sequences that share a prefix (gfx950).
//
//   out[b][h] = sum_t softmax_t(scale q[b][h].K[t]) V[t],  t < L_b,
// the first s_b = min(shared_lens[b], L_b) tokens of sequence b being those of the
// first sequence of its group, whose table they are read through; the rest is
// read through b's own table.  L_b <= 0 writes zeros.  Sums are fp32.
#include <algorithm>
#include <climits>
#include <cmath>

#include "../device_api.hpp"
#include "common.hpp"

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
    const int shared = lead < 0 ? 0 : max(0, min(p.shared_lens[b], L));
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

}  // namespace

namespace dev {

uint64_t attn_shared_scratch_bytes(int32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) {
    return 256;
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
