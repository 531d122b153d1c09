// gguf_epilogue.hpp -- what the linear layer does with a product before it
// leaves the kernel, on gfx950.
//
//   y[m, n] = cast( act( sum_k x[m, k] W[n, k] + bias[n] ) * mul[m, n] + residual[m, n] )
//
// in fp32 up to the one rounding of the cast (nearest, ties to even).  The
// product kernels take their output as a type of its own: `float *` is the
// plain fp32 matrix of the GEMM entries, an Epilogue the linear layer's y; the
// sums before it are the same.  mul and residual have y's type and may be y
// itself: the thread that stores an element read it before.
//
// Fused because the product is the only thing that has it at hand: a second
// pass reads and writes every element again and costs a launch (2 to 3 us,
// the time of a small decode product).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gollek {

enum ElementType : int { kF32 = 0, kF16 = 1, kBF16 = 30 };  // ggml type ids
enum Activation : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4 };

struct Epilogue {
    void *y;
    const float *bias;     // N floats, or nullptr
    const void *mul;       // or nullptr
    const void *residual;  // or nullptr
    int64_t y_stride, mul_stride, residual_stride;  // elements between rows
    int act, type;
    bool vec4;  // every matrix's rows allow loads and stores of four elements
};

inline Epilogue make_epilogue(void *y, const float *bias, const void *mul, const void *residual, int64_t y_stride,
                              int64_t mul_stride, int64_t residual_stride, int act, int type) {
    const uintptr_t size = type == kF32 ? 4 : 2;
    uintptr_t low = reinterpret_cast<uintptr_t>(y) | (uintptr_t)y_stride * size;
    if (mul != nullptr) low |= reinterpret_cast<uintptr_t>(mul) | (uintptr_t)mul_stride * size;
    if (residual != nullptr) low |= reinterpret_cast<uintptr_t>(residual) | (uintptr_t)residual_stride * size;
    return {y,        bias, mul,  residual, y_stride, mul_stride, residual_stride,
            act,      type, (low & (4 * size - 1)) == 0};
}

// v / (1 + exp(-s v)) at s v: exp overflows to infinity past 88, which leaves -0.
__device__ __forceinline__ float gated(float v, float s) { return v / (1.0f + expf(-s)); }

__device__ __forceinline__ float activate(int act, float v) {
    switch (act) {
    case kActRelu: return v < 0.0f ? 0.0f : v;  // (NaN stays)
    case kActSilu: return gated(v, v);
    case kActGelu: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    // 0.5 (1 + tanh(z)) is 1 / (1 + exp(-2 z))
    case kActGeluTanh: return gated(v, 1.5957691216057308f * (v + 0.044715f * v * v * v));
    default: return v;
    }
}

__device__ __forceinline__ float load_element(const void *p, int type, int64_t i) {
    if (type == kF32) return static_cast<const float *>(p)[i];
    if (type == kF16) return (float)static_cast<const _Float16 *>(p)[i];
    return __uint_as_float((uint32_t)static_cast<const uint16_t *>(p)[i] << 16);
}
__device__ __forceinline__ void store_element(void *p, int type, int64_t i, float v) {
    if (type == kF32) static_cast<float *>(p)[i] = v;
    else if (type == kF16) static_cast<_Float16 *>(p)[i] = (_Float16)v;
    else static_cast<__bf16 *>(p)[i] = (__bf16)v;
}

// Element (m, n) of an output with N columns.
__device__ __forceinline__ void put(float *y, int64_t m, int64_t n, int64_t N, float v) { y[m * N + n] = v; }
__device__ __forceinline__ void put(const Epilogue &e, int64_t m, int64_t n, int64_t, float v) {
    if (e.bias != nullptr) v += e.bias[n];
    v = activate(e.act, v);
    if (e.mul != nullptr) v *= load_element(e.mul, e.type, m * e.mul_stride + n);
    if (e.residual != nullptr) v += load_element(e.residual, e.type, m * e.residual_stride + n);
    store_element(e.y, e.type, m * e.y_stride + n, v);
}

// Elements (m, n .. n + 3), those past column N - 1 left out.
__device__ __forceinline__ void put4(const Epilogue &e, int64_t m, int64_t n, int64_t N, float4 v) {
    const float a[4] = {v.x, v.y, v.z, v.w};
    for (int i = 0; i < 4 && n + i < N; i++) put(e, m, n + i, N, a[i]);
}

// Where split `split` of a product with `mn` outputs leaves its sums: a plain
// matrix takes split 0 itself, an epilogue waits for all of them.
__device__ __forceinline__ float *split_output(float *y, float *part, int split, int64_t mn) {
    return split == 0 ? y : part + (split - 1) * mn;
}
__device__ __forceinline__ float *split_output(const Epilogue &, float *part, int split, int64_t mn) {
    return part + split * mn;
}

template <class OUT>
constexpr bool kHasEpilogue = false;
template <>
inline constexpr bool kHasEpilogue<Epilogue> = true;

// Host side: workspace bytes left for the S - 1 partials that a split plan
// counts (an epilogue's split 0 takes one more), and whether a product's
// splits can be added four floats at a time.
template <class OUT>
size_t split_bytes(const float *workspace, size_t bytes, int M, int N) {
    if (workspace == nullptr) return 0;
    const size_t first = kHasEpilogue<OUT> ? (size_t)M * N * sizeof(float) : 0;
    return bytes > first ? bytes - first : 0;
}
inline bool splits_aligned(const float *y, const float *workspace, int M, int N) {
    return ((int64_t)M * N) % 4 == 0 &&
           ((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(y)) & 15u) == 0;
}
inline bool splits_aligned(const Epilogue &, const float *workspace, int M, int N) {
    return ((int64_t)M * N) % 4 == 0 && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0;
}

}  // namespace gollek
