// Low-rank adapters of many requests beside a shared projection (gfx950):
//   y[t] = bf16(base[t] + scale_a (x[t] A_a^T) B_a^T),  a = adapter_ids[t],
// A_a [slices * rank][k] and B_a [n][rank] bf16; column n takes the rank values
// of its slice.  A token without an adapter keeps base.  The low-rank values pass
// through memory of the caller's, in fp32; y is rounded once.
#include <algorithm>
#include <climits>

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
    int ends[4];
};

// One wave a low-rank value.
__global__ __launch_bounds__(256) void lora_shrink_simple(LoraParams p) {
    const int lane = threadIdx.x & 63;
    const int t = blockIdx.x, r = blockIdx.y * 4 + (threadIdx.x >> 6);
    const int id = p.ids[t];
    if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.adapters) || r >= p.rows) return;
    const uint16_t* x = p.x + static_cast<size_t>(t) * p.k;
    const uint16_t* a = p.a + (static_cast<size_t>(id) * p.rows + r) * p.k;
    float sum = 0.0f;
    for (int i = lane; i < p.k; i += 64) sum += bf16_bits_to_f32(x[i]) * bf16_bits_to_f32(a[i]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) p.low[static_cast<size_t>(t) * p.rows + r] = sum;
}

// One thread an output.
__global__ __launch_bounds__(256) void lora_expand_simple(LoraParams p) {
    const int t = blockIdx.x, c = blockIdx.y * 256 + threadIdx.x;
    if (c >= p.n) return;
    const size_t at = static_cast<size_t>(t) * p.n + c;
    const int id = p.ids[t];
    if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.adapters)) {
        p.y[at] = p.base[at];
        return;
    }
    int s = 0;
    while (c >= p.ends[s]) ++s;
    const float* low = p.low + static_cast<size_t>(t) * p.rows + s * p.rank;
    const uint16_t* b = p.b + (static_cast<size_t>(id) * p.n + c) * p.rank;
    float sum = 0.0f;
    for (int r = 0; r < p.rank; ++r) sum += low[r] * bf16_bits_to_f32(b[r]);
    const float scale = p.scales != nullptr ? p.scales[id] : 1.0f;
    p.y[at] = static_cast<uint16_t>(f32_to_bf16_bits(bf16_bits_to_f32(p.base[at]) + scale * sum));
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
    hipLaunchKernelGGL(lora_shrink_simple, dim3(p.m, (p.rows + 3) / 4), dim3(256), 0, s, p);
    KCMM_HIP_CHECK(hipGetLastError(), err);
    hipLaunchKernelGGL(lora_expand_simple, dim3(p.m, (p.n + 255) / 256), dim3(256), 0, s, p);
    KCMM_HIP_CHECK(hipGetLastError(), err);
    return true;
}

}  // namespace dev
}  // namespace kcmm
