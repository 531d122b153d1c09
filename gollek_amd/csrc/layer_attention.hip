// layer_attention.hip -- attention of one new token a sequence over a paged cache
// of keys and values, on gfx950.
//
//   s_j = scale * q . k_j [softcap * tanh(s_j / softcap)]
//   out = sum_j exp(s_j) v_j / (sum_j exp(s_j) [+ exp(sink)])
//
// in one pass: m the largest s so far, l = sum exp(s_j - m), o = sum exp(s_j - m) v_j,
// the last two scaled by exp(m_old - m) whenever m grows.
#include <hip/hip_runtime.h>

#include "layer_kernels.hpp"

namespace gollek {
namespace {

constexpr int kWaves = 4;

// One workgroup a query head; its waves take every fourth token.
__global__ __launch_bounds__(64 * kWaves) void attend_kernel(AttendArgs a) {
    __shared__ float part_m[kWaves], part_l[kWaves], part_o[kWaves][256];
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, dim = a.kv.head_dim;
    const int head = (int)blockIdx.x % a.q_heads, kv_head = head / (a.q_heads / a.kv.kv_heads);
    const int64_t sequence = blockIdx.x / a.q_heads;
    const int64_t table = a.max_pages << a.kv.page_shift;
    const int64_t length = min((int64_t)max(a.lengths[sequence], 0), table);
    const int64_t begin = a.window > 0 && length > a.window ? length - a.window : 0;
    const float ninf = -__builtin_inff();

    float q[4], o[4] = {};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = lane + 64 * i;
        q[i] = d < dim ? load_element(a.q, a.kv.type, sequence * a.q_stride + (int64_t)head * dim + d) : 0.0f;
    }
    float m = ninf, l = 0.0f;
    for (int64_t j = begin + wave; j < length; j += kWaves) {
        const int64_t page = a.page_table[sequence * a.max_pages + (j >> a.kv.page_shift)];
        if (page < 0 || page >= a.kv.pages) continue;
        const int64_t slot = j & ((1 << a.kv.page_shift) - 1);
        const int64_t at = (((page * a.kv.kv_heads + kv_head) << a.kv.page_shift) + slot) * dim;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < dim) s += q[i] * load_element(a.kv.k, a.kv.type, at + lane + 64 * i);
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) s += __shfl_xor(s, x);
        s *= a.scale;
        if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
        const float most = fmaxf(m, s), base = most == ninf ? 0.0f : most;
        const float keep = expf(m - base), p = expf(s - base);
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            o[i] *= keep;
            if (lane + 64 * i < dim) o[i] += p * load_element(a.kv.v, a.kv.type, at + lane + 64 * i);
        }
        m = most;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) part_o[wave][lane + 64 * i] = o[i];
    if (lane == 0) part_m[wave] = m, part_l[wave] = l;
    __syncthreads();
    float most = a.sinks != nullptr ? a.sinks[head] : ninf;
    const float sink = most;
    for (int w = 0; w < kWaves; w++) most = fmaxf(most, part_m[w]);
    const float base = most == ninf ? 0.0f : most;
    float total = a.sinks != nullptr ? expf(sink - base) : 0.0f;
    for (int w = 0; w < kWaves; w++) total += part_l[w] * expf(part_m[w] - base);
    for (int d = (int)threadIdx.x; d < dim; d += 64 * kWaves) {
        float v = 0.0f;
        for (int w = 0; w < kWaves; w++) v += part_o[w][d] * expf(part_m[w] - base);
        store_element(a.out, a.out_type, sequence * a.out_stride + (int64_t)head * dim + d, total > 0.0f || total != total ? v / total : 0.0f);
    }
}

}  // namespace

size_t attend_workspace_bytes(const KvPages &, int, int, int64_t) { return 0; }

hipError_t launch_attend(const AttendArgs &a, uint8_t *, hipStream_t stream) {
    hipLaunchKernelGGL(attend_kernel, dim3((unsigned)(a.sequences * a.q_heads)), dim3(64 * kWaves), 0, stream, a);
    return hipGetLastError();
}

}  // namespace gollek
