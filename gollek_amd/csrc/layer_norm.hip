// layer_norm.hip -- the norms around a block, on gfx950.
//
//   b = post ? N(x) * post : x;  h = residual + scale * gate * b  -> hidden
//   y = N(h) * weight + bias;  N(v) = v / sqrt(mean(v^2) + eps), or of v - mean(v)
//
// One workgroup a row; the row stays in registers in fp32 from the first load to
// the last store, so x and the residual are read once and nothing is read back.
#include <hip/hip_runtime.h>

#include "layer_kernels.hpp"

namespace gollek {
namespace {

// The sum of v over a workgroup of WAVES waves, in every thread.
template <int WAVES>
__device__ __forceinline__ float block_sum(float v, float *lds) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    if constexpr (WAVES > 1) {
        __syncthreads();  // (the sum before is read)
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < WAVES; w++) v += lds[w];
    }
    return v;
}

// Elements c * 64 * WAVES + thread of a row, c < PER.
template <int WAVES, int PER>
__global__ __launch_bounds__(64 * WAVES) void norm_kernel(NormArgs a) {
    __shared__ float lds[WAVES];
    const int64_t row = blockIdx.x;
    float h[PER];
    const auto each = [&](auto f) {
#pragma unroll
        for (int c = 0; c < PER; c++) {
            const int i = c * 64 * WAVES + (int)threadIdx.x;
            if (i < a.cols) f(c, i);
        }
    };
    const auto normalise = [&] {  // h <- N(h)
        float sum = 0.0f;
        if (a.layer) {
            each([&](int c, int) { sum += h[c]; });
            const float mean = block_sum<WAVES>(sum, lds) / (float)a.cols;
            each([&](int c, int) { h[c] -= mean; });
            sum = 0.0f;
        }
        each([&](int c, int) { sum += h[c] * h[c]; });
        const float r = 1.0f / sqrtf(block_sum<WAVES>(sum, lds) / (float)a.cols + a.eps);
        each([&](int c, int) { h[c] *= r; });
    };
    each([&](int c, int i) { h[c] = load_element(a.x, a.x_type, row * a.x_stride + i); });
    if (a.post != nullptr) {
        normalise();
        each([&](int c, int i) { h[c] *= a.post[i]; });
    }
    each([&](int c, int i) {
        h[c] *= a.scale;
        if (a.gate != nullptr) h[c] *= a.gate[i];
        if (a.residual != nullptr) h[c] += load_element(a.residual, a.hidden_type, row * a.residual_stride + i);
        if (a.hidden != nullptr) store_element(a.hidden, a.hidden_type, row * a.hidden_stride + i, h[c]);
    });
    if (a.y == nullptr) return;
    normalise();
    each([&](int c, int i) {
        float v = a.weight != nullptr ? h[c] * a.weight[i] : h[c];
        if (a.bias != nullptr) v += a.bias[i];
        store_element(a.y, a.y_type, row * a.y_stride + i, v);
    });
}

}  // namespace

hipError_t launch_norm(const NormArgs &a, hipStream_t stream) {
    const dim3 grid((unsigned)a.rows);
    if (a.cols <= 4096) hipLaunchKernelGGL((norm_kernel<4, 16>), grid, dim3(256), 0, stream, a);
    else if (a.cols <= 16384) hipLaunchKernelGGL((norm_kernel<16, 16>), grid, dim3(1024), 0, stream, a);
    else hipLaunchKernelGGL((norm_kernel<16, 64>), grid, dim3(1024), 0, stream, a);
    return hipGetLastError();
}

}  // namespace gollek
