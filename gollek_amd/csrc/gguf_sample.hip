// gguf_sample.hip -- one token per row of lm_head logits, on gfx950.
//
// Row of V logits l, largest m; tokens ordered by logit, equal ones by index:
//   w_i = exp((l_i - m) / T)          (T <= 0: the first token alone)
//   kept: the first top_k; of these the shortest prefix whose mass (sum of w)
//         reaches top_p of theirs; of these w_i >= min_p
//   token = the first index, in the vocabulary's order, whose cumulative kept
//         mass exceeds u times the kept mass.
// -inf and NaN logits are no tokens.  Every filter keeps a prefix of the order,
// so the kept set is a threshold (key, index).
//
// Masses are 64-bit integers, w in units of 2^-S with V 2^S < 2^62 (2^-44 for a
// vocabulary of 128k to 256k): integer sums do not depend on the order of the
// additions, so neither the split of a row over workgroups nor atomics change a
// token, and their rounding (2^-45 a token) is far below what fp32 sums would
// lose at the borders of top_p and u.
#include <hip/hip_runtime.h>

#include "gguf_kernels.hpp"

namespace gollek {
namespace {

typedef unsigned long long u64;

// A logit as an unsigned integer of the same order; 0 for what is no token.
__device__ __forceinline__ uint32_t logit_key(float l) {
    if (!(l > -__builtin_inff())) return 0;
    const uint32_t b = __float_as_uint(l + 0.0f);  // (-0 is 0)
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k);
}

// Weights of a row.
struct Scale {
    float m;       // the largest logit
    double inv_t;  // 1 / T
    int shift;     // S
    __device__ __forceinline__ double weight(float l) const {
        if (m == __builtin_inff()) return l == m ? 1.0 : 0.0;
        return exp(((double)l - (double)m) * inv_t);
    }
    __device__ __forceinline__ u64 fixed(double w) const { return (u64)(__builtin_ldexp(w, shift) + 0.5); }
};

struct SampleArgs {
    const void *logits;
    int64_t stride;
    int type, vocab, shift;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *tokens, *kept;
    float *probs;
};

constexpr int kThreads = 1024, kWaves = kThreads / 64;

struct Border {  // kept: key > this one, or the same key at an index up to this one
    uint32_t key;
    int index;
    __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= index); }
};

// What a row asks for, in range.
struct Wish {
    double inv_t, top_p, min_p, u;
    int top_k;
    bool has_p;
};
__device__ __forceinline__ Wish row_wish(const SampleArgs &a, int row) {
    Wish w;
    const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
    w.top_k = a.top_k != nullptr ? a.top_k[row] : 0;
    if (!(t > 0.0f)) w.top_k = 1;
    if (w.top_k <= 0 || w.top_k > a.vocab) w.top_k = a.vocab;
    w.inv_t = t > 0.0f ? 1.0 / (double)t : 1.0;
    const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
    w.has_p = p < 1.0f;
    w.top_p = p;
    if (w.has_p && !(p > 0.0f)) {  // nothing reaches past the first token
        w.top_k = 1;
        w.has_p = false;
    }
    const float mp = a.min_p != nullptr ? a.min_p[row] : 0.0f;
    w.min_p = mp > 1.0f ? 1.0 : mp > 0.0f ? (double)mp : 0.0;
    const float u = a.u[row];
    w.u = u >= 1.0f ? 1.0 - 0x1p-24 : u > 0.0f ? (double)u : 0.0;
    return w;
}

struct RowLds {
    u64 mass[256];
    uint32_t count[256];
    u64 part[kWaves + 1];
    uint32_t digit;
    u64 before_mass;
    uint32_t before_count;
    int found;
};

// The sum over the workgroup, in every thread.
template <class V>
__device__ V block_sum(V v, RowLds &s) {
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = (u64)v;
    __syncthreads();
    V t = 0;
    for (int w = 0; w < kWaves; w++) t += (V)s.part[w];
    return t;
}

// The border of the elements within `in` that are the first `count` in order
// (by_mass: the shortest prefix whose mass is not below `target`): a digit of
// the key at a time, from the top; then the index among equal keys.
__device__ Border select(const SampleArgs &a, int64_t base, const Scale &sc, Border in, bool by_mass, uint32_t count,
                         double target, RowLds &s) {
    uint32_t prefix = 0, seen = 0;
    u64 mass = 0;
    uint32_t ties = 0;
    for (int at = 24; at >= 0; at -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) {
            s.mass[threadIdx.x] = 0;
            s.count[threadIdx.x] = 0;
        }
        __syncthreads();
        for (int i = (int)threadIdx.x; i < a.vocab; i += kThreads) {
            const float l = load_element(a.logits, a.type, base + i);
            const uint32_t k = logit_key(l);
            if (k == 0 || !in.keeps(k, i) || (at < 24 && (k >> (at + 8)) != (prefix >> (at + 8)))) continue;
            const uint32_t d = (k >> at) & 255u;
            atomicAdd(&s.count[d], 1u);  // LDS
            if (by_mass) atomicAdd(&s.mass[d], sc.fixed(sc.weight(l)));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t c = seen;
            u64 m = mass;
            int d = 255;
            for (; d > 0; d--) {
                if (by_mass ? !((double)(m + s.mass[d]) < target) : c + s.count[d] >= count) break;
                c += s.count[d];
                m += s.mass[d];
            }
            s.digit = (uint32_t)d;
            s.before_count = c;
            s.before_mass = m;
        }
        __syncthreads();
        prefix |= s.digit << at;
        seen = s.before_count;
        mass = s.before_mass;
        ties = s.count[s.digit];
    }
    // `r` of the `ties` equal keys
    uint32_t r;
    if (by_mass) {
        const u64 w = sc.fixed(sc.weight(key_logit(prefix)));
        u64 lo = 1, hi = ties;  // the smallest r whose mass is not below the target
        while (lo < hi) {
            const u64 mid = (lo + hi) / 2;
            if ((double)(mass + mid * w) < target) lo = mid + 1;
            else hi = mid;
        }
        r = (uint32_t)lo;
    } else {
        r = count - seen;
    }
    if (r >= ties) return Border{prefix, 0x7FFFFFFF};
    // the index of the r-th of them: kThreads indexes at a time
    if (threadIdx.x == 0) s.found = 0x7FFFFFFF;
    uint32_t had = 0;
    for (int i0 = 0; i0 < a.vocab; i0 += kThreads) {
        const int i = i0 + (int)threadIdx.x;
        bool is = false;
        if (i < a.vocab) {
            const uint32_t k = logit_key(load_element(a.logits, a.type, base + i));
            is = k == prefix && in.keeps(k, i);
        }
        const u64 who = __ballot(is);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6] = (u64)__builtin_popcountll(who);
        __syncthreads();
        uint32_t before = had, all = had;
        for (int w = 0; w < kWaves; w++) {
            if (w < (int)(threadIdx.x >> 6)) before += (uint32_t)s.part[w];
            all += (uint32_t)s.part[w];
        }
        const uint32_t place = before + (uint32_t)__builtin_popcountll(who & ((1ull << (threadIdx.x & 63)) - 1ull)) + 1u;
        if (is && place == r) s.found = i;
        had = all;
        if (had >= r) break;  // (the same in every thread)
    }
    __syncthreads();
    return Border{prefix, s.found};
}

// One workgroup per row.
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ RowLds s;
    __shared__ float wave_max[kWaves];
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x;
    const int64_t base = (int64_t)row * a.stride;
    const Wish wish = row_wish(a, row);

    float m = -__builtin_inff();
    for (int i = tid; i < a.vocab; i += kThreads) m = fmaxf(m, load_element(a.logits, a.type, base + i));
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    if ((tid & 63) == 0) wave_max[tid >> 6] = m;
    __syncthreads();
    for (int w = 0; w < kWaves; w++) m = fmaxf(m, wave_max[w]);
    if (!(m > -__builtin_inff())) {  // no token at all
        if (tid == 0) {
            a.tokens[row] = -1;
            if (a.probs != nullptr) a.probs[row] = 0.0f;
            if (a.kept != nullptr) a.kept[row] = 0;
        }
        return;
    }
    const Scale sc = {m, wish.inv_t, a.shift};

    // Mass and number of the tokens within a border that min_p keeps.
    auto sum = [&](Border in, double min_p, u64 &mass, uint32_t &n) {
        u64 t = 0;
        uint32_t c = 0;
        for (int i = tid; i < a.vocab; i += kThreads) {
            const float l = load_element(a.logits, a.type, base + i);
            const uint32_t k = logit_key(l);
            if (k == 0 || !in.keeps(k, i)) continue;
            const double w = sc.weight(l);
            if (!(w >= min_p)) continue;
            t += sc.fixed(w);
            c++;
        }
        mass = block_sum(t, s);
        n = block_sum(c, s);
    };
    Border border = {0, 0x7FFFFFFF};
    u64 total;
    uint32_t kept;
    sum(border, 0.0, total, kept);
    if ((uint32_t)wish.top_k < kept) {
        border = select(a, base, sc, border, false, (uint32_t)wish.top_k, 0.0, s);
        sum(border, 0.0, total, kept);
    }
    if (wish.has_p) {
        border = select(a, base, sc, border, true, 0, wish.top_p * (double)total, s);
    }
    sum(border, wish.min_p, total, kept);

    // The draw, kThreads indexes at a time.
    const double target = wish.u * (double)total;
    u64 had = 0;
    for (int i0 = 0; i0 < a.vocab; i0 += kThreads) {
        const int i = i0 + tid;
        u64 f = 0;
        double w = 0.0;
        if (i < a.vocab) {
            const float l = load_element(a.logits, a.type, base + i);
            const uint32_t k = logit_key(l);
            if (k != 0 && border.keeps(k, i)) {
                w = sc.weight(l);
                if (w >= wish.min_p) f = sc.fixed(w);
            }
        }
        u64 cum = f;  // inclusive over the wave
        for (int d = 1; d < 64; d <<= 1) {
            const u64 o = __shfl_up(cum, d);
            if ((tid & 63) >= d) cum += o;
        }
        __syncthreads();
        if ((tid & 63) == 63) s.part[tid >> 6] = cum;
        __syncthreads();
        u64 before = had, all = had;
        for (int v = 0; v < kWaves; v++) {
            if (v < (tid >> 6)) before += s.part[v];
            all += s.part[v];
        }
        cum += before;
        if (f > 0 && (double)cum > target && !((double)(cum - f) > target)) {  // one thread, once
            a.tokens[row] = i;
            if (a.probs != nullptr) a.probs[row] = (float)(__builtin_ldexp(w, a.shift) / (double)total);
            if (a.kept != nullptr) a.kept[row] = (int32_t)kept;
        }
        had = all;
        if ((double)had > target) break;
    }
}

}  // namespace

size_t sample_workspace_bytes(int rows, int vocab) {
    (void)rows;
    (void)vocab;
    return 0;
}

hipError_t launch_sample(const void *logits, int logits_type, int rows, int vocab, int64_t stride,
                         const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                         const float *u, int32_t *tokens, float *probs, int32_t *kept, uint8_t *workspace,
                         hipStream_t stream) {
    (void)workspace;
    if (rows <= 0) return hipSuccess;
    int bits = 1;
    while ((1ll << bits) <= vocab) bits++;
    const SampleArgs a = {logits, stride, logits_type, vocab,  62 - bits, temperature,
                          top_p,  min_p,  u,           top_k,  tokens,    kept,        probs};
    hipLaunchKernelGGL(sample_row_kernel, dim3((unsigned)rows), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace gollek
