// layer_heads.hip -- rotary positions, and new keys and values into a paged cache,
// on gfx950.
//
// Per head: h <- h / sqrt(mean(h^2) + eps) * norm (optional), then every pair of its
// first `dims` elements turns by the token's position:
//   (a, b) <- magnitude * (a cos t - b sin t, b cos t + a sin t),  t = position * f_i.
// The angle is position * turns_i in 64 bits with its whole revolutions taken off:
// fp32 would be off by 2^-24 of the position, 0.006 revolutions at 100000.  What is left, at
// most half a revolution, goes to sine and cosine as an fp32 number and what that lost: in one
// number sines next to half a revolution would be off by 2^-23.3, and random heads by 3.4e-8 in
// place of 2.9e-8.
//
// A wave works on heads of one token.  Its lanes compute one sine and cosine each (all
// heads of a token have the same angles) and share them through LDS; then a group of
// lanes takes a head, a lane V pairs of it: V neighbours and their V partners, two loads
// of up to 16 bytes at 16-bit elements.  Many tokens: a wave takes all heads of its token,
// one group after the other; few: the heads are dealt to more waves.
//
// Bound by bytes where there are many tokens: 4096 tokens of 32 heads of 128 rotated 11.9
// us (67 MB), 4096 with 8 + 8 heads of keys and values into a cache 21 to 23 (101 MB; a
// wave a head, its sines its own, 82).  One token, 3.4 us, is a launch and the chain
// position, page, store; everything else is loaded before it.
#include <hip/hip_runtime.h>

#include "gguf_kernels.hpp"  // device_cus
#include "layer_kernels.hpp"

namespace gollek {
namespace {

constexpr int kWaves = 4, kMostPairs = 128;

// V elements of SIZE bytes, at any alignment of the element.
template <int SIZE, int V>
struct Run {
    alignas(SIZE * V < 4 ? SIZE * V : 4) uint8_t bytes[SIZE * V];
    __device__ __forceinline__ void load(const void *p, int64_t i) {
        __builtin_memcpy(bytes, static_cast<const uint8_t *>(p) + i * SIZE, sizeof(bytes));
    }
    __device__ __forceinline__ void store(void *p, int64_t i) const {
        __builtin_memcpy(static_cast<uint8_t *>(p) + i * SIZE, bytes, sizeof(bytes));
    }
    __device__ __forceinline__ void get(float *v, int type) const {
        if constexpr (SIZE == 4) {
            __builtin_memcpy(v, bytes, sizeof(bytes));
        } else {
            uint16_t w[V];
            __builtin_memcpy(w, bytes, sizeof(bytes));
            if (type == kBF16) {
#pragma unroll
                for (int j = 0; j < V; j++) v[j] = __uint_as_float((uint32_t)w[j] << 16);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) v[j] = (float)__builtin_bit_cast(_Float16, w[j]);
            }
        }
    }
    __device__ __forceinline__ void set(const float *v, int type) {
        if constexpr (SIZE == 4) {
            __builtin_memcpy(bytes, v, sizeof(bytes));
        } else {
            uint16_t w[V];
            if (type == kBF16) {
#pragma unroll
                for (int j = 0; j < V; j++) w[j] = __builtin_bit_cast(uint16_t, (__bf16)v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) w[j] = __builtin_bit_cast(uint16_t, (_Float16)v[j]);
            }
            __builtin_memcpy(bytes, w, sizeof(bytes));
        }
    }
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
// The sum over each group of `lanes` (a power of two), in all of them.
__device__ __forceinline__ float group_sum(float v, int lanes) {
    if (lanes > 1) v = dpp_add<0xB1>(v);   // quad_perm [1, 0, 3, 2]
    if (lanes > 2) v = dpp_add<0x4E>(v);   // quad_perm [2, 3, 0, 1]
    if (lanes > 4) v = dpp_add<0x141>(v);  // row_half_mirror
    if (lanes > 8) v = dpp_add<0x140>(v);  // row_mirror
    if (lanes > 16) v += __shfl_xor(v, 16);
    if (lanes > 32) v += __shfl_xor(v, 32);
    return v;
}

struct HeadsPlan {
    int lanes;   // of a head, a power of two
    int slices;  // waves of a token
};

// IN, OUT: element sizes.  V pairs a lane, in NS places of the head (2 for heads of more
// than 64 lanes' pairs).  CACHE: keys and values go to a cache, else queries alone.
template <int IN, int OUT, int V, int NS, bool CACHE>
__global__ __launch_bounds__(64 * kWaves) void heads_kernel(HeadsArgs a, HeadsPlan plan) {
    __shared__ float2 turns[kWaves][kMostPairs];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t unit = (int64_t)blockIdx.x * kWaves + wave;
    const bool in = unit < a.tokens * plan.slices;
    // (a wave past the last token loads what the first one does, and leaves)
    const int64_t t = in ? unit / plan.slices : 0;
    const int slice = in ? (int)(unit - t * plan.slices) : 0;
    const int kv_heads = CACHE ? a.kv.kv_heads : 0, heads = a.q_heads + 2 * kv_heads;
    const int dim = a.head_dim, dims = a.rope.dims, pairs = dim / 2;
    // everything that waits for nothing is loaded first: a decoded token's call is a chain
    // of loads, position to page to place, and the angles on the way
    const int64_t position = a.positions[t];
    int64_t sequence = -1, page = -1;
    if constexpr (CACHE) {
        sequence = a.sequence != nullptr ? a.sequence[t] : a.first + t;
    }
    // this lane's pairs: p .. p + V - 1; their first and second elements stand at
    // e0 and e1 .. (half), or together from e0 on (interleaved, or behind what turns)
    const int groups = 64 / plan.lanes, mine = lane % plan.lanes;
    int e0[NS], e1[NS];
    bool has[NS], turned[NS];
    Run<4, V> qn[NS][2], kn[NS][2];
#pragma unroll
    for (int n = 0; n < NS; n++) {
        const int p = V * (mine + 64 * n);
        has[n] = p < pairs;
        turned[n] = p < dims / 2;
        const bool half = turned[n] && !a.rope.interleaved;
        e0[n] = half ? p : 2 * p;
        e1[n] = half ? p + dims / 2 : 2 * p + V;
        if (!has[n]) continue;
        if (a.q_norm != nullptr) qn[n][0].load(a.q_norm, e0[n]), qn[n][1].load(a.q_norm, e1[n]);
        if (a.k_norm != nullptr) kn[n][0].load(a.k_norm, e0[n]), kn[n][1].load(a.k_norm, e1[n]);
    }
    // the token's rows (taken here: chosen by lane from the arguments themselves, the
    // pointers would go through scratch memory)
    const uint8_t *q_row = static_cast<const uint8_t *>(a.q) + t * a.q_stride * IN;
    const uint8_t *k_row = nullptr, *v_row = nullptr;
    if constexpr (CACHE) {
        k_row = static_cast<const uint8_t *>(a.k) + t * a.k_stride * IN;
        v_row = static_cast<const uint8_t *>(a.v) + t * a.v_stride * IN;
    }
    Run<IN, V> x[NS][2];
    const auto fetch = [&](int head) {
        const uint8_t *from = q_row + (int64_t)head * dim * IN;
        if (CACHE && head >= a.q_heads) {
            const bool key = head < a.q_heads + kv_heads;
            from = (key ? k_row : v_row) + (int64_t)(head - a.q_heads - (key ? 0 : kv_heads)) * dim * IN;
        }
#pragma unroll
        for (int n = 0; n < NS; n++)
            if (has[n]) x[n][0].load(from, e0[n]), x[n][1].load(from, e1[n]);
    };
    int head = slice * groups + lane / plan.lanes;
    if (head < heads) fetch(head);
    double angle[2];
#pragma unroll
    for (int n = 0; n < 2; n++) angle[n] = lane + 64 * n < dims / 2 ? a.rope.turns[lane + 64 * n] : 0.0;

    // the token's place in the cache: of head 0, in elements (-1: nowhere)
    int64_t place = -1;
    bool padding = false;
    if constexpr (CACHE) {
        const int64_t column = position >> a.kv.page_shift;
        padding = position < 0 || sequence < 0 || sequence >= a.sequences;
        if (!padding && column < a.max_pages) page = a.page_table[sequence * a.max_pages + column];
    }
#pragma unroll
    for (int n = 0; n < 2; n++) {
        if (lane + 64 * n >= dims / 2) continue;
        const double turn = (double)position * angle[n], part = turn - rint(turn);
        const float near = (float)part, rest = (float)(2.0 * M_PI * (part - (double)near));
        float s, c;
        sincospif(2.0f * near, &s, &c);
        turns[wave][lane + 64 * n] = make_float2(a.rope.magnitude * fmaf(-s, rest, c), a.rope.magnitude * fmaf(c, rest, s));
    }
    __syncthreads();
    if (!in || padding) return;
    if constexpr (CACHE) {
        const int64_t slot = position & ((1 << a.kv.page_shift) - 1);
        if (page >= 0 && page < a.kv.pages) place = (((page * kv_heads) << a.kv.page_shift) + slot) * dim;
    }
    float2 cs[NS][V];
#pragma unroll
    for (int n = 0; n < NS; n++)
#pragma unroll
        for (int j = 0; j < V; j++)
            cs[n][j] = turned[n] ? turns[wave][V * (mine + 64 * n) + j] : make_float2(1.0f, 0.0f);

    const int64_t v_from_k = static_cast<uint8_t *>(a.kv.v) - static_cast<uint8_t *>(a.kv.k);
    const int step = plan.slices * groups;
    const int rounds = (heads - slice * groups + step - 1) / step;  // (of the wave; its last may lack heads)
    for (int i = 0; i < rounds; i++, head += step) {
        float u[NS][2][V];
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < NS; n++) {
            x[n][0].get(u[n][0], a.type);
            x[n][1].get(u[n][1], a.type);
#pragma unroll
            for (int j = 0; j < V; j++)
                if (has[n]) sum += u[n][0][j] * u[n][0][j] + u[n][1][j] * u[n][1][j];
        }
        if (head + step < heads) fetch(head + step);
        const bool query = head < a.q_heads, key = !query && head < a.q_heads + kv_heads;
        if (a.q_norm != nullptr || a.k_norm != nullptr) {
            const float r = 1.0f / sqrtf(group_sum(sum, plan.lanes) / (float)dim + a.eps);
            if ((query && a.q_norm != nullptr) || (key && a.k_norm != nullptr)) {
#pragma unroll
                for (int n = 0; n < NS; n++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float q[V], k[V];
                        qn[n][h].get(q, kF32);
                        kn[n][h].get(k, kF32);
#pragma unroll
                        for (int j = 0; j < V; j++) u[n][h][j] *= r * (query ? q[j] : k[j]);
                    }
            }
        }
        if (head >= heads || (!query && place < 0)) continue;
        uint8_t *to = static_cast<uint8_t *>(a.q_out);
        int64_t at = t * a.q_out_stride + (int64_t)head * dim;
        if (CACHE && !query) {
            to = static_cast<uint8_t *>(a.kv.k) + (key ? 0 : v_from_k);
            at = place + ((int64_t)(head - a.q_heads - (key ? 0 : kv_heads)) << a.kv.page_shift) * dim;
        }
#pragma unroll
        for (int n = 0; n < NS; n++) {
            if (!has[n]) continue;
            float y[2][V];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < V; j++) y[h][j] = u[n][h][j];
            if (turned[n] && (!CACHE || query || key)) {
                // pair j: first and second element
                if (a.rope.interleaved) {
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        float &p = y[2 * j / V][2 * j % V], &q = y[(2 * j + 1) / V][(2 * j + 1) % V];
                        const float w = p * cs[n][j].x - q * cs[n][j].y;
                        q = q * cs[n][j].x + p * cs[n][j].y;
                        p = w;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const float w = y[0][j] * cs[n][j].x - y[1][j] * cs[n][j].y;
                        y[1][j] = y[1][j] * cs[n][j].x + y[0][j] * cs[n][j].y;
                        y[0][j] = w;
                    }
                }
            }
            Run<OUT, V> out[2];
            out[0].set(y[0], a.out_type);
            out[1].set(y[1], a.out_type);
            out[0].store(to, at + e0[n]);
            out[1].store(to, at + e1[n]);
        }
    }
}

template <int IN, int OUT, bool CACHE>
hipError_t launch(const HeadsArgs &a, hipStream_t stream) {
    const int heads = a.q_heads + (CACHE ? 2 * a.kv.kv_heads : 0), pairs = a.head_dim / 2, turned = a.rope.dims / 2;
    // V divides what turns and the whole, so a lane's pairs are of one kind
    const auto fits = [&](int v) { return pairs % v == 0 && turned % v == 0; };
    const int v = fits(8) ? 8 : fits(4) ? 4 : fits(2) ? 2 : 1;
    HeadsPlan p = {1, 1};
    while (p.lanes < 64 && p.lanes * v < pairs) p.lanes *= 2;
    const int groups = 64 / p.lanes, rounds = (heads + groups - 1) / groups;
    const int64_t waves = (int64_t)device_cus() * 16;  // four a SIMD
    p.slices = (int)(a.tokens >= waves ? 1 : (waves + a.tokens - 1) / a.tokens < rounds ? (waves + a.tokens - 1) / a.tokens : rounds);
    const int64_t blocks = (a.tokens * p.slices + kWaves - 1) / kWaves;
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * kWaves), 0, stream, a, p);
        return hipGetLastError();
    };
    if (v == 8) return go(heads_kernel<IN, OUT, 8, 1, CACHE>);
    if (v == 4) return go(heads_kernel<IN, OUT, 4, 1, CACHE>);
    if (v == 2) return go(heads_kernel<IN, OUT, 2, 1, CACHE>);
    return go(heads_kernel<IN, OUT, 1, 2, CACHE>);
}

}  // namespace

hipError_t launch_heads(const HeadsArgs &all, hipStream_t stream) {
    // A grid has at most 2^32 threads in all: more than kMostTokens take several.
    constexpr int64_t kMostTokens = (int64_t)1 << 25;
    HeadsArgs a = all;
    const auto moved = [&](const void *p, int64_t stride, int type) -> const void * {
        return p == nullptr ? nullptr : static_cast<const uint8_t *>(p) + a.first * stride * (type == kF32 ? 4 : 2);
    };
    for (a.first = 0; a.first < all.tokens; a.first += kMostTokens) {
        a.tokens = all.tokens - a.first < kMostTokens ? all.tokens - a.first : kMostTokens;
        a.q = moved(all.q, a.q_stride, a.type);
        a.k = moved(all.k, a.k_stride, a.type);
        a.v = moved(all.v, a.v_stride, a.type);
        a.q_out = const_cast<void *>(moved(all.q_out, a.q_out_stride, a.out_type));
        a.positions = all.positions + a.first;
        if (all.sequence != nullptr) a.sequence = all.sequence + a.first;
        const bool wide = a.type == kF32;
        const hipError_t e = a.kv.k != nullptr ? (wide ? launch<4, 2, true>(a, stream) : launch<2, 2, true>(a, stream))
                                               : (wide ? launch<4, 4, false>(a, stream) : launch<2, 2, false>(a, stream));
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace gollek
