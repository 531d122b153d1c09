// layer_heads.hip -- rotary positions, and new keys and values into a paged cache,
// on gfx950.
//
// Per head: h <- h / sqrt(mean(h^2) + eps) * norm (optional), then every pair of its
// first `dims` elements turns by the token's position:
//   (a, b) <- magnitude * (a cos t - b sin t, b cos t + a sin t),  t = position * f_i.
// The angle is position * turns_i in 64 bits with its whole revolutions taken off:
// fp32 would be off by 2^-24 of the position, 0.006 revolutions at 100000.
#include <hip/hip_runtime.h>

#include "layer_kernels.hpp"

namespace gollek {
namespace {

// One wave a head of a token; lane l has pairs l and l + 64.
__global__ __launch_bounds__(256) void heads_kernel(HeadsArgs a) {
    const int lane = (int)threadIdx.x & 63;
    const int kv_heads = a.kv.k != nullptr ? a.kv.kv_heads : 0, heads = a.q_heads + 2 * kv_heads, dim = a.head_dim;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), t = unit / heads;
    if (t >= a.tokens) return;
    int head = (int)(unit - t * heads);
    const int64_t position = a.positions[t];
    int part = 0;  // q, k, v
    if (head >= a.q_heads) head -= a.q_heads, part = 1;
    if (part == 1 && head >= kv_heads) head -= kv_heads, part = 2;

    const void *const src = part == 0 ? a.q : part == 1 ? a.k : a.v;
    const int64_t from = t * (part == 0 ? a.q_stride : part == 1 ? a.k_stride : a.v_stride) + (int64_t)head * dim;
    void *dst = a.q_out;
    int64_t to = t * a.q_out_stride + (int64_t)head * dim;
    if (kv_heads != 0) {
        const int64_t sequence = a.sequence != nullptr ? a.sequence[t] : t;
        if (position < 0 || sequence < 0 || sequence >= a.sequences) return;  // padding
        if (part != 0) {
            const int64_t column = position >> a.kv.page_shift, slot = position & ((1 << a.kv.page_shift) - 1);
            if (column >= a.max_pages) return;
            const int64_t page = a.page_table[sequence * a.max_pages + column];
            if (page < 0 || page >= a.kv.pages) return;
            dst = part == 1 ? a.kv.k : a.kv.v;
            to = (((page * kv_heads + head) << a.kv.page_shift) + slot) * dim;
        }
    }
    const float *const norm = part == 0 ? a.q_norm : part == 1 ? a.k_norm : nullptr;
    const int dims = part == 2 ? 0 : a.rope.dims;

    float x[2][2];
    int e[2][2];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int p = lane + 64 * j;
        if (p >= dim / 2) continue;
        const bool half = p < dims / 2 && !a.rope.interleaved;
        e[j][0] = half ? p : 2 * p;
        e[j][1] = half ? p + dims / 2 : 2 * p + 1;
        for (int i = 0; i < 2; i++) {
            x[j][i] = load_element(src, a.type, from + e[j][i]);
            sum += x[j][i] * x[j][i];
        }
    }
    float r = 1.0f;
    if (norm != nullptr) {
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
        r = 1.0f / sqrtf(sum / (float)dim + a.eps);
    }
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int p = lane + 64 * j;
        if (p >= dim / 2) continue;
        float u = x[j][0], v = x[j][1];
        if (norm != nullptr) u *= r * norm[e[j][0]], v *= r * norm[e[j][1]];
        if (p < dims / 2) {
            const double turn = (double)position * a.rope.turns[p];
            float s, c;
            sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
            s *= a.rope.magnitude, c *= a.rope.magnitude;
            const float w = u * c - v * s;
            v = v * c + u * s;
            u = w;
        }
        store_element(dst, a.out_type, to + e[j][0], u);
        store_element(dst, a.out_type, to + e[j][1], v);
    }
}

}  // namespace

hipError_t launch_heads(const HeadsArgs &a, hipStream_t stream) {
    const int64_t heads = a.q_heads + (a.kv.k != nullptr ? 2 * a.kv.kv_heads : 0), blocks = (a.tokens * heads + 3) / 4;
    if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
    hipLaunchKernelGGL(heads_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace gollek
