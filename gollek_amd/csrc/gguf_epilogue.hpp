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
// the time of a small decode product).  Measured: Q4_K M = 2048, 14336 x 4096 with
// SiLU, mul and bf16 out 344 us, the product alone with fp32 out 338; one token of
// Q8_0 1024 x 4096 with bias and residual 4.9 in a graph of launches, the mat-vec 4.6.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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
    bool vec;  // every matrix's rows start on 16-byte boundaries
};

inline Epilogue make_epilogue(void *y, const float *bias, const void *mul, const void *residual, int64_t y_stride,
                              int64_t mul_stride, int64_t residual_stride, int act, int type) {
    const uintptr_t size = type == kF32 ? 4 : 2;
    uintptr_t low = reinterpret_cast<uintptr_t>(y) | (uintptr_t)y_stride * size;
    if (mul != nullptr) low |= reinterpret_cast<uintptr_t>(mul) | (uintptr_t)mul_stride * size;
    if (residual != nullptr) low |= reinterpret_cast<uintptr_t>(residual) | (uintptr_t)residual_stride * size;
    return {y,        bias, mul,  residual, y_stride, mul_stride, residual_stride,
            act,      type, (low & 15u) == 0};
}

// v / (1 + exp(-s)); past 88 exp(-s) overflows to infinity, which leaves -0.
// FAST, for results that are rounded to 16 bits: exp as 2^(s log2 e) by the
// hardware's instruction, whose argument's rounding makes it 2^-24 |s| off,
// and a reciprocal good to 2^-23: a tenth of fp16's half step up to |s| = 400
// (beyond it the result is below fp16's range).  A quarter of the exact form's
// instructions, which cost a 96 x 256 tile 4 us.
template <bool FAST>
__device__ __forceinline__ float gated(float v, float s) {
    if constexpr (FAST)
        return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * s));
    return v / (1.0f + expf(-s));
}

// v Phi(v) without 1 + erf, which cancels below 0 (4 % off at v = -5, 0 at -6):
//   Phi(-a) = t (1/2 + c1 s + .. + c7 s^7) exp(-a^2 / 2),  t = 1 / (1 + 0.3 a),  s = 1 - t = 0.3 a t,
// the coefficients a minimax fit of the relative error over a in [0, 14]: 2^-22.7;
// in fp32 3 units of 2^-23 from v = -1 on and 6 at -3; below it is exp's argument,
// a^2 / 2, that rounds, as v's own last bit would.  At 16, where a stops, exp has
// left fp32's range.  Serves fp32 results too: the library's erfc is as exact and
// cost a 96 x 256 tile's products 4 to 8 %.
__device__ __forceinline__ float gelu(float v) {
    const float a = fminf(fabsf(v), 16.0f), pa = 0.3f * a;
    const float t = __builtin_amdgcn_rcpf(1.0f + pa), s = pa * t;
    constexpr float kTerm[8] = {0.5f,           -0.829805851f, 0.618176758f,  -0.0820174515f,
                                -0.131090671f, -0.0126647931f, 0.0927853063f, -0.0357543267f};
    float q = kTerm[7];
#pragma unroll
    for (int k = 6; k >= 0; k--) q = __builtin_fmaf(q, s, kTerm[k]);
    q = q * t * __builtin_amdgcn_exp2f(-0.72134752044448170f * a * a);
    return v * (v < 0.0f ? q : 1.0f - q);
}

template <bool FAST>
__device__ __forceinline__ float activate(int act, float v) {
    switch (act) {
    case kActRelu: return v < 0.0f ? 0.0f : v;  // (NaN stays)
    case kActSilu: return gated<FAST>(v, v);
    case kActGelu: return gelu(v);
    // 0.5 (1 + tanh(z)) is 1 / (1 + exp(-2 z))
    case kActGeluTanh: return gated<FAST>(v, 1.5957691216057308f * (v + 0.044715f * v * v * v));
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

template <class OUT>
constexpr bool kHasEpilogue = false;
template <>
inline constexpr bool kHasEpilogue<Epilogue> = true;

// The type a kernel takes for OUT.  Launches name it: a plain output deduced from
// an argument, or passed on as float *, would lose its __restrict__.
typedef float *__restrict__ PlainOut;
template <class OUT>
using KernelOut = std::conditional_t<kHasEpilogue<OUT>, OUT, PlainOut>;

// Element (m, n) of an output with N columns.
__device__ __forceinline__ void put(float *y, int64_t m, int64_t n, int64_t N, float v) { y[m * N + n] = v; }
__device__ __forceinline__ void put(const Epilogue &e, int64_t m, int64_t n, int64_t, float v) {
    if (e.bias != nullptr) v += e.bias[n];
    v = e.type == kF32 ? activate<false>(e.act, v) : activate<true>(e.act, v);
    if (e.mul != nullptr) v *= load_element(e.mul, e.type, m * e.mul_stride + n);
    if (e.residual != nullptr) v += load_element(e.residual, e.type, m * e.residual_stride + n);
    store_element(e.y, e.type, m * e.y_stride + n, v);
}

// The same in two steps: what an element needs beside its sum, loaded while the
// product still runs (a load behind it costs the small products 1 us), and the rest.
struct Ahead {
    float bias, mul, residual;
};
struct NoAhead {};
__device__ __forceinline__ NoAhead load_ahead(float *, bool, int64_t, int64_t) { return {}; }
__device__ __forceinline__ Ahead load_ahead(const Epilogue &e, bool in, int64_t m, int64_t n) {
    Ahead a = {0.0f, 1.0f, 0.0f};
    if (in && e.bias != nullptr) a.bias = e.bias[n];
    if (in && e.mul != nullptr) a.mul = load_element(e.mul, e.type, m * e.mul_stride + n);
    if (in && e.residual != nullptr) a.residual = load_element(e.residual, e.type, m * e.residual_stride + n);
    return a;
}
__device__ __forceinline__ void put(float *y, int64_t m, int64_t n, int64_t N, float v, NoAhead) { y[m * N + n] = v; }
__device__ __forceinline__ void put(const Epilogue &e, int64_t m, int64_t n, int64_t, float v, const Ahead &a) {
    if (e.bias != nullptr) v += a.bias;
    v = e.type == kF32 ? activate<false>(e.act, v) : activate<true>(e.act, v);
    if (e.mul != nullptr) v *= a.mul;
    if (e.residual != nullptr) v += a.residual;
    store_element(e.y, e.type, m * e.y_stride + n, v);
}

// Elements in W words: 16 bytes of them (Elements), or four (Quad).
template <int TYPE, int W>
struct Words {
    static constexpr int kSize = TYPE == kF32 ? 4 : 2, kCount = 4 * W / kSize;
    typedef uint32_t words __attribute__((ext_vector_type(W)));
    words bits;
    __device__ __forceinline__ void load(const void *p, int64_t i) {
        bits = *reinterpret_cast<const words *>(static_cast<const uint8_t *>(p) + i * kSize);
    }
    __device__ __forceinline__ void store(void *p, int64_t i) const {
        *reinterpret_cast<words *>(static_cast<uint8_t *>(p) + i * kSize) = bits;
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (TYPE == kF32) return __uint_as_float(bits[j]);
        const uint32_t w = bits[j >> 1];
        if constexpr (TYPE == kBF16) return __uint_as_float((j & 1) ? w & 0xFFFF0000u : w << 16);
        return (float)__builtin_bit_cast(_Float16, (uint16_t)((j & 1) ? w >> 16 : w & 0xFFFFu));
    }
    __device__ __forceinline__ void set(const float *v) {
#pragma unroll
        for (int j = 0; j < W; j++) {
            if constexpr (TYPE == kF32) {
                bits[j] = __float_as_uint(v[j]);
            } else if constexpr (TYPE == kBF16) {
                typedef __bf16 b2 __attribute__((ext_vector_type(2)));
                bits[j] = __builtin_bit_cast(uint32_t, b2{(__bf16)v[2 * j], (__bf16)v[2 * j + 1]});
            } else {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                bits[j] = __builtin_bit_cast(uint32_t, h2{(_Float16)v[2 * j], (_Float16)v[2 * j + 1]});
            }
        }
    }
};
template <int TYPE>
using Elements = Words<TYPE, 4>;
template <int TYPE>
using Quad = Words<TYPE, TYPE == kF32 ? 4 : 2>;

// The activations of C values (one uniform branch for all of them).
template <bool FAST, int C>
__device__ __forceinline__ void activate_all(int act, float (&v)[C]) {
    switch (act) {
#define GOLLEK_ACT(A)                                                                 \
    case A:                                                                           \
        _Pragma("unroll") for (int j = 0; j < C; j++) v[j] = activate<FAST>(A, v[j]); \
        break
        GOLLEK_ACT(kActRelu);
        GOLLEK_ACT(kActSilu);
        GOLLEK_ACT(kActGelu);
        GOLLEK_ACT(kActGeluTanh);
#undef GOLLEK_ACT
    default: break;
    }
}

// A ROWS x COLS tile of fp32 sums, row-major in LDS with rows kTilePitch<COLS>
// floats apart, through the epilogue.  A thread takes 16 bytes of a row at a
// time, in rounds of THREADS of them; the mul and residual of up to four rounds
// (a batch) are loaded together, a batch before it is used: the first by
// tile_ahead, which may stand anywhere before, the next while one is computed.
// (Q4_K M = 2048, 14336 x 4096 with SiLU and mul: 464 us element by element,
// straight from the accumulators, where every load waited behind the store before
// it; 378 in rows; 344 with the loads a batch ahead and activations FAST.)
template <int COLS>
constexpr int kTilePitch = COLS + 4;

template <int ROWS, int COLS, int THREADS, int TYPE>
struct TileRounds {
    static constexpr int kCount = Elements<TYPE>::kCount, kAcross = COLS / kCount;  // vectors of a row
    static constexpr int kStep = THREADS / kAcross;                                 // rows of a round
    static constexpr int kRounds = (ROWS + kStep - 1) / kStep;
    static constexpr int kBatch = kRounds < 4 ? kRounds : 4;
    static_assert(THREADS % kAcross == 0, "whole rows a round");
};

template <int ROWS, int COLS, int THREADS>
struct TileAhead {
    static constexpr int kBatch = TileRounds<ROWS, COLS, THREADS, kF32>::kBatch;  // (F32 has the most rounds)
    Elements<kF32> mul[kBatch], residual[kBatch];
};

// Rounds i0 .. i0 + kBatch - 1 of a thread.
template <int ROWS, int COLS, int THREADS, int TYPE, class V, int B>
__device__ __forceinline__ void tile_fetch(const Epilogue &e, int m0, int n0, int M, int N, int tid, int i0, V (&mul)[B],
                                           V (&residual)[B]) {
    using R = TileRounds<ROWS, COLS, THREADS, TYPE>;
    constexpr int size = Elements<TYPE>::kSize;
    const int n = n0 + R::kCount * (tid % R::kAcross), row = tid / R::kAcross;
#pragma unroll
    for (int i = 0; i < R::kBatch; i++) {
        const int r = row + (i0 + i) * R::kStep;
        if (r >= ROWS || m0 + r >= M || !e.vec || n + R::kCount > N) continue;
        if (e.mul != nullptr) mul[i].load(e.mul, ((int64_t)(m0 + r) * e.mul_stride + n) * size / V::kSize);
        if (e.residual != nullptr)
            residual[i].load(e.residual, ((int64_t)(m0 + r) * e.residual_stride + n) * size / V::kSize);
    }
}

template <int ROWS, int COLS, int THREADS>
__device__ __forceinline__ void tile_ahead(const Epilogue &e, int m0, int n0, int M, int N, int tid,
                                           TileAhead<ROWS, COLS, THREADS> &a) {
    if (e.type == kF32) tile_fetch<ROWS, COLS, THREADS, kF32>(e, m0, n0, M, N, tid, 0, a.mul, a.residual);
    else tile_fetch<ROWS, COLS, THREADS, kF16>(e, m0, n0, M, N, tid, 0, a.mul, a.residual);  // (as BF16)
}

template <int ROWS, int COLS, int THREADS, int TYPE>
__device__ __forceinline__ void put_tile_as(const Epilogue &e, const float *tile, int m0, int n0, int M, int N, int tid,
                                            const TileAhead<ROWS, COLS, THREADS> &first) {
    using V = Elements<TYPE>;
    using R = TileRounds<ROWS, COLS, THREADS, TYPE>;
    constexpr int C = R::kCount, B = R::kBatch;
    const int col = C * (tid % R::kAcross), row = tid / R::kAcross, n = n0 + col;
    const bool whole = e.vec && n + C <= N;
    float bias[C];
    if (whole && e.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < C; j++) bias[j] = e.bias[n + j];
    }
    V mul[2][B], residual[2][B];
#pragma unroll
    for (int i = 0; i < B; i++) {
        mul[0][i].bits = first.mul[i].bits;
        residual[0][i].bits = first.residual[i].bits;
    }
#pragma unroll
    for (int b = 0; b * B < R::kRounds; b++) {
        if ((b + 1) * B < R::kRounds)
            tile_fetch<ROWS, COLS, THREADS, TYPE>(e, m0, n0, M, N, tid, (b + 1) * B, mul[(b + 1) & 1],
                                                  residual[(b + 1) & 1]);
#pragma unroll
        for (int i = 0; i < B; i++) {
            const int r = row + (b * B + i) * R::kStep;
            if (r >= ROWS || m0 + r >= M) continue;
            const float *const from = tile + r * kTilePitch<COLS> + col;
            float v[C];
#pragma unroll
            for (int j = 0; j < C; j += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(from + j);
                v[j] = f.x, v[j + 1] = f.y, v[j + 2] = f.z, v[j + 3] = f.w;
            }
            if (whole) {
                if (e.bias != nullptr) {
#pragma unroll
                    for (int j = 0; j < C; j++) v[j] += bias[j];
                }
                activate_all<TYPE != kF32>(e.act, v);
                if (e.mul != nullptr) {
#pragma unroll
                    for (int j = 0; j < C; j++) v[j] *= mul[b & 1][i].get(j);
                }
                if (e.residual != nullptr) {
#pragma unroll
                    for (int j = 0; j < C; j++) v[j] += residual[b & 1][i].get(j);
                }
                V out;
                out.set(v);
                out.store(e.y, (int64_t)(m0 + r) * e.y_stride + n);
            } else {
                for (int j = 0; j < C && n + j < N; j++) put(e, m0 + r, n + j, N, from[j]);
            }
        }
    }
}

// The tile stands in LDS (a barrier after its writes); `first` from tile_ahead.
template <int ROWS, int COLS, int THREADS>
__device__ __forceinline__ void put_tile(const Epilogue &e, const float *tile, int m0, int n0, int M, int N, int tid,
                                         const TileAhead<ROWS, COLS, THREADS> &first) {
    if (e.type == kF32) put_tile_as<ROWS, COLS, THREADS, kF32>(e, tile, m0, n0, M, N, tid, first);
    else if (e.type == kF16) put_tile_as<ROWS, COLS, THREADS, kF16>(e, tile, m0, n0, M, N, tid, first);
    else put_tile_as<ROWS, COLS, THREADS, kBF16>(e, tile, m0, n0, M, N, tid, first);
}

// Where split `split` of a product with `mn` outputs leaves its sums: a plain
// matrix takes split 0 itself, an epilogue waits for all of them.
__device__ __forceinline__ float *split_output(float *y, float *part, int split, int64_t mn) {
    return split == 0 ? y : part + (split - 1) * mn;
}
__device__ __forceinline__ float *split_output(const Epilogue &, float *part, int split, int64_t mn) {
    return part + split * mn;
}

// Host side: workspace bytes left for the S - 1 partials that a split plan
// counts (an epilogue's split 0 takes one more), and whether a product's
// splits can be added (a plain one's four floats at a time).
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
inline bool splits_aligned(const Epilogue &, const float *workspace, int, int) {
    return (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0;
}

}  // namespace gollek
