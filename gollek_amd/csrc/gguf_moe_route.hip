// gguf_moe_route.hip -- routing to experts with a balancing bias, groups and
// weights as the model wants them, on gfx950.
//
// Per token, over its E router logits l:
//   p = softmax(l) or 1 / (1 + exp(-l));  c = p + bias (what is chosen by);
//   a group (E / G neighbours) is worth the sum of its one or two largest c;
//   the top_groups worthiest groups stay, and of their experts the top_k with
//   the largest c are taken, ties to the lower index, NaN above everything;
//   weight = p (not c) of each, over their sum if asked (and the sum is > 0),
//   times scale.
// Scores, sums and comparisons are in double: p differs between neighbouring
// fp32 logits by less than fp32 resolves (near 1 for the sigmoid), and c is
// compared after a sum.  The exps in double cost 1M a call of 8192 x 128, 1.5 us
// of the chip.
//
// One wave per token (lane l holds experts l, l + 64, ...), so nothing
// waits at a workgroup barrier.  The largest of 64 lanes' keys is six DPP maxima
// of the keys' upper halves; only lanes that agree there compare the lower ones.
// Bound by the rounds, which depend on each other: 8192 x 128 bf16, top 8 9.5 us (2.6
// MB, 0.5 us of the card's copy rate), 256 x 256 with groups 8.3, one token 4.2 on the
// GPU.  (Plain routing by moe_topk_kernel, which counts ranks and rounds as the
// reference does: 8192 x 128 62.6, one token 10.4.)
#include <hip/hip_runtime.h>

#include "gguf_kernels.hpp"

namespace gollek {
namespace {

typedef unsigned long long u64;

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
// The largest of the wave's values, in every lane (0 is the identity).
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, dpp<0x111, 0xF>(v));  // row_shr 1, 2, 4, 8: lane 15 of a row has its row's
    v = max(v, dpp<0x112, 0xF>(v));
    v = max(v, dpp<0x114, 0xF>(v));
    v = max(v, dpp<0x118, 0xF>(v));
    v = max(v, dpp<0x142, 0xA>(v));  // row_bcast 15, 31: lane 63 has the wave's
    v = max(v, dpp<0x143, 0xC>(v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ double shfl_xor_f64(double v, int mask) {
    const u64 b = __builtin_bit_cast(u64, v);
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)b, mask), hi = (uint32_t)__shfl_xor((int)(b >> 32), mask);
    return __builtin_bit_cast(double, ((u64)hi << 32) | lo);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += shfl_xor_f64(v, m);
    return v;
}

// Unsigned order of doubles: -inf .. inf, then NaN; every key above 0.
__device__ __forceinline__ u64 order_key(double v) {
    if (v != v) return ~0ull;
    const u64 b = __builtin_bit_cast(u64, v + 0.0);  // (-0 is 0)
    return (b >> 63) ? ~b : b | (1ull << 63);
}

// a, b <- the two larger of a >= b and x >= y, by key.
struct Pair {
    u64 a, b;
    __device__ __forceinline__ void add(u64 x) {
        if (x > a) {
            b = a;
            a = x;
        } else if (x > b) b = x;
    }
};

struct RouteArgs {
    const void *logits;
    const float *bias;
    int32_t *ids;
    float *weights;
    int tokens, experts, top_k, groups, top_groups, group_top, type;
    bool sigmoid, renormalize;
    float scale;
};

// PER experts per lane; WAVES tokens per workgroup.  GROUPS: some groups are
// left out (the call has fewer top_groups than groups).
template <int PER, int WAVES, bool GROUPS>
__global__ __launch_bounds__(64 * WAVES) void moe_route_kernel(RouteArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t route_lds[];
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int t = (int)blockIdx.x * WAVES + wave;
    if (t >= a.tokens) return;  // (a wave on its own: no barrier follows)
    const int E = a.experts, K = a.top_k;
    double *const ps = reinterpret_cast<double *>(route_lds) + (size_t)wave * (GROUPS ? 2 : 1) * E;  // p of every expert
    double *const cs = ps + E;                                                                       // c, for the groups
    const int64_t row = (int64_t)t * E;

    float l[PER];
    float mx = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int e = lane + 64 * j;
        l[j] = e < E ? load_element(a.logits, a.type, row + e) : -__builtin_inff();
        mx = fmaxf(mx, l[j]);
    }
    double p[PER];
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < PER; j++) p[j] = 1.0 / (1.0 + exp(-(double)l[j]));
    } else {
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) mx = fmaxf(mx, __shfl_xor(mx, m));
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            p[j] = exp((double)l[j] - (double)mx);
            if (lane + 64 * j < E) s += p[j];
        }
        const double over = 1.0 / wave_sum(s);
#pragma unroll
        for (int j = 0; j < PER; j++) p[j] *= over;
    }
    u64 key[PER];
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int e = lane + 64 * j;
        key[j] = 0;
        if (e < E) {
            const double c = a.bias != nullptr ? p[j] + (double)a.bias[e] : p[j];
            key[j] = order_key(c);
            ps[e] = p[j];
            if constexpr (GROUPS) cs[e] = c;
        }
    }
    __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses complete in order)

    if constexpr (GROUPS) {
        // L lanes (a power of two) per group collect its two largest c and merge.
        const int size = E / a.groups;
        int L = 64;
        while (L * a.groups > 64) L >>= 1;
        const int g = lane / L, i0 = lane - g * L;
        Pair best = {0, 0};
        if (g < a.groups)
            for (int i = i0; i < size; i += L) best.add(order_key(cs[g * size + i]));
        for (int m = 1; m < L; m <<= 1) {
            const u64 x = __shfl_xor(best.a, m), y = __shfl_xor(best.b, m);
            best.add(x);
            best.add(y);
        }
        auto value = [](u64 k) {  // the double of a key
            if (k == ~0ull) return __builtin_nan("");
            return __builtin_bit_cast(double, (k >> 63) ? k ^ (1ull << 63) : ~k);
        };
        u64 worth = 0;
        if (g < a.groups)
            worth = a.group_top == 2 && best.b != 0 ? order_key(value(best.a) + value(best.b)) : best.a;
        // A group's rank: the groups ahead of it.
        int rank = 0;
        for (int o = 0; o < a.groups; o++) {
            const u64 other = __shfl(worth, o * L);
            rank += other > worth || (other == worth && o < g);
        }
        const u64 kept = __ballot(g < a.groups && rank < a.top_groups);  // every lane of a kept group
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int e = lane + 64 * j;
            if (e < E && ((kept >> ((e / size) * L)) & 1) == 0) key[j] = 0;
        }
    }

    // The top_k: each round takes the wave's largest key (lowest index) out.
    u64 mine = 0;   // this lane's largest key ...
    int at = 0;     // ... and its j (the lowest)
    auto look = [&] {
        mine = 0;
        at = 0;
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (key[j] > mine) {
                mine = key[j];
                at = j;
            }
    };
    look();
    const bool few = K <= 64;  // lane r keeps rank r
    int id = 0;
    for (int r = 0; r < K; r++) {
        const uint32_t hi = (uint32_t)(mine >> 32);
        u64 who = __ballot(hi == wave_max(hi));
        int winner;
        if (__builtin_popcountll(who) == 1) {
            winner = __builtin_ctzll(who);
        } else {
            const bool in = (who >> lane) & 1;
            const uint32_t lo = in ? (uint32_t)mine : 0u;
            const uint32_t top = wave_max(lo);
            who = __ballot(in && lo == top);
            // equal keys: the lowest index, e = lane + 64 at
            const bool tie = (who >> lane) & 1;
            const uint32_t low = wave_max(tie ? 0xFFFFFFFFu - (uint32_t)(lane + 64 * at) : 0u);
            winner = (int)((0xFFFFFFFFu - low) & 63u);
        }
        const int e = winner + 64 * __builtin_amdgcn_readlane(at, winner);
        if (few) id = lane == r ? e : id;
        else if (lane == 0) a.ids[(int64_t)t * K + r] = e;
        if (lane == winner) {
#pragma unroll
            for (int j = 0; j < PER; j++)
                if (j == at) key[j] = 0;
            look();
        }
    }
    if (!few) __threadfence_block();  // lane 0's ids
    double sum = 0.0;
    for (int r = lane; r < K; r += 64) sum += ps[few ? id : a.ids[(int64_t)t * K + r]];
    sum = wave_sum(sum);
    const double over = a.renormalize && sum > 0.0 ? sum : 1.0;
    for (int r = lane; r < K; r += 64) {
        const int e = few ? id : a.ids[(int64_t)t * K + r];
        if (few) a.ids[(int64_t)t * K + r] = e;
        a.weights[(int64_t)t * K + r] = (float)(ps[e] / over * (double)a.scale);
    }
}

template <int PER, int WAVES>
hipError_t launch(const RouteArgs &a, hipStream_t stream) {
    const dim3 grid((unsigned)((a.tokens + WAVES - 1) / WAVES)), block(64 * WAVES);
    const size_t row = (size_t)a.experts * sizeof(double) * WAVES;
    if (a.top_groups < a.groups)
        hipLaunchKernelGGL((moe_route_kernel<PER, WAVES, true>), grid, block, 2 * row, stream, a);
    else hipLaunchKernelGGL((moe_route_kernel<PER, WAVES, false>), grid, block, row, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_moe_expert_route(const void *logits, int logits_type, int T, int E, const float *bias, bool sigmoid,
                                   int groups, int top_groups, int group_top, int top_k, bool renormalize, float scale,
                                   int32_t *ids, float *weights, hipStream_t stream) {
    if (T <= 0) return hipSuccess;
    const RouteArgs a = {logits, bias,   ids,        weights,   T,           E,       top_k,
                         groups, top_groups, group_top, logits_type, sigmoid, renormalize, scale};
    if (E <= 64) return launch<1, 4>(a, stream);
    if (E <= 128) return launch<2, 4>(a, stream);
    if (E <= 256) return launch<4, 4>(a, stream);
    if (E <= 512) return launch<8, 4>(a, stream);
    if (E <= 1024) return launch<16, 2>(a, stream);
    if (E <= 4096) return launch<64, 1>(a, stream);
    return hipErrorInvalidValue;
}

}  // namespace gollek
