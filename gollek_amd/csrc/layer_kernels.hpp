// layer_kernels.hpp -- host-side launchers of the kernels between a decoder
// layer's products: norms, rotary positions, the paged key-value cache and its
// attention.  Asynchronous on `stream`, device pointers; arguments are checked in
// the C-ABI layer (layer_capi.hip).  Strides in elements.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "gguf_epilogue.hpp"  // element types

namespace gollek {

// b = post ? N(x) * post : x;  h = residual + scale * gate * b;  y = N(h) * weight + bias.
struct NormArgs {
    const void *x, *residual;
    void *hidden, *y;
    const float *post, *gate, *weight, *bias;
    int64_t x_stride, residual_stride, hidden_stride, y_stride;
    int64_t rows;
    int cols, x_type, hidden_type, y_type;
    bool layer;
    float scale, eps;
};
hipError_t launch_norm(const NormArgs &a, hipStream_t stream);

// Rotary tables: turns (revolutions a position) of each pair in 64 bits, on the device.
struct RopeTable {
    const double *turns;
    int dims;  // rotated elements of a head (0: none)
    bool interleaved;
    float magnitude;
};

// The paged cache, each array (pages, kv_heads, page_size, head_dim).
struct KvPages {
    void *k, *v;
    int64_t pages;
    int page_shift, kv_heads, head_dim, type;
};

// Heads of new tokens: q to a matrix, k and v to a cache (kv.k nullptr: q alone).
struct HeadsArgs {
    const void *q, *k, *v;
    void *q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const float *q_norm, *k_norm;
    float eps;
    RopeTable rope;
    KvPages kv;
    const int32_t *positions, *sequence, *page_table;
    int64_t sequences, max_pages;
    int64_t tokens;
    int64_t first;  // the launch's first token's number in the call (sequence nullptr: its sequence)
    int q_heads, head_dim, type, out_type;
};
hipError_t launch_heads(const HeadsArgs &a, hipStream_t stream);

struct AttendArgs {
    KvPages kv;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    const int32_t *lengths, *page_table;
    const float *sinks;
    int64_t max_pages;
    int sequences, q_heads, out_type, window;
    float scale, softcap;
};
size_t attend_workspace_bytes(const KvPages &kv, int sequences, int q_heads, int64_t max_pages);
hipError_t launch_attend(const AttendArgs &a, uint8_t *workspace, hipStream_t stream);

}  // namespace gollek
