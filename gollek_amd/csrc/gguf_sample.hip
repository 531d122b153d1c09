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
// Masses are 64-bit integers, w in units of 2^-S with S <= 50 and V 2^S < 2^62 (2^-44 for a
// vocabulary of 128k to 256k): integer sums do not depend on the order of the
// additions, so neither the split of a row over workgroups nor atomics change a
// token, and their rounding (2^-45 a token) is far below what fp32 sums would
// lose at the borders of top_p and u.
//
// A vocabulary of up to 16384 is one workgroup's, in its registers (the end of this
// file).  A longer row is cut into slabs of 256 tokens, sixteen of them a chunk, and
// the chunks dealt to workgroups; four launches:
//   1 the largest logit of every slab (reads the row);
//   2 rows with a filter: a histogram (tokens, and mass for top_p) over 512 bins
//     of l, linear from the largest logit down to where weights round to 0 (or to
//     the least logit); rows without: every chunk's kept mass;
//   3 from the histogram, the bin in which the filter's border falls; the tokens
//     of the bins down to it are collected, or, where that is more than 4096,
//     those of the border's bin alone and the chunks' mass above it;
//   4 one workgroup per row: the collected tokens sorted, the border in them, the
//     draw: the chunk that the random number falls into, then the token.
// A top_k of up to 64, and to as many as the slabs that hold a token, goes without 2 and 3:
// its tokens lie above the top_k-th largest slab maximum, in those slabs alone,
// which the last launch reads itself.  (Every row passes every launch, since the
// settings are on the device; with many rows 3 is two, a plan and the collection.)
// A row whose border bin holds more than 4096 tokens (equal logits, a
// temperature of 30), or whose top_p border depends on a top_k border that far
// down, is computed by the last workgroup alone, digit by digit over the row: one
// row with top_k 5000 and top_p 0.9 222 us at 32000 tokens, 629 at 128256 and 1223
// at 262144 (top_k 5000 alone 34 to 37).
//
// Bound by the launches' dependence and, for many rows, by the weights in double:
// one row of 128256 fp32 logits with top_k 40 and top_p 18.8 us, 64 of them with
// mixed filters 53 to 56 (33 MB, 6.4 us of the card's copy rate), 16 rows of 32000 bf16
// without a filter 19.7.
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

// Weights of a row: w = 2^t, t = (l - m) log2(e) / T, as 2^f of t's fraction by
// its Taylor series (|f| <= 1/2: the term left out is below 2^-52) times 2^n.
// (20 instructions in double; the library's exp and its conversion to an integer
// cost 64 rows of 128256 3 us more.)
struct Scale {
    float m;       // the largest logit
    double rate;   // log2(e) / T
    double unit;   // 2^S
    __device__ __forceinline__ Scale(float top, double inv_t, int shift)
        : m(top), rate(inv_t * 1.4426950408889634), unit(__builtin_ldexp(1.0, shift)) {}
    __device__ __forceinline__ double weight(float l) const {
        if (m == __builtin_inff()) return l == m ? 1.0 : 0.0;
        const double t = __builtin_fmax(((double)l - (double)m) * rate, -2000.0);
        const double n = __builtin_rint(t), f = t - n;
        // ln(2)^k / k!
        constexpr double kTerm[13] = {1.0,
                                      6.9314718055994531e-01,
                                      2.4022650695910072e-01,
                                      5.5504108664821580e-02,
                                      9.6181291076284772e-03,
                                      1.3333558146428443e-03,
                                      1.5403530393381609e-04,
                                      1.5252733804059841e-05,
                                      1.3215486790144309e-06,
                                      1.0178086009239699e-07,
                                      7.0549116208011233e-09,
                                      4.4455382718708114e-10,
                                      2.5678435993488202e-11};
        double p = kTerm[12];
#pragma unroll
        for (int k = 11; k >= 0; k--) p = __builtin_fma(p, f, kTerm[k]);
        return __builtin_ldexp(p, (int)n);
    }
    // w in units of 2^-S, rounded: w 2^S <= 2^50 stands in the low bits of 2^52 more.
    __device__ __forceinline__ u64 fixed(double w) const {
        return __builtin_bit_cast(u64, __builtin_fma(w, unit, 0x1p52)) & ((1ull << 52) - 1);
    }
};

struct SampleArgs {
    const void *logits;
    int64_t stride;
    int type, vocab, shift;
    bool vec4;  // rows allow loads of four logits
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *tokens, *kept;
    float *probs;
};

constexpr int kThreads = 1024, kWaves = kThreads / 64;  // of the last launch
constexpr int kScan = 256;                              // of the others
constexpr int kChunk = 4096, kBins = 512, kList = 4096;
constexpr int kChunkSlabs = 16;
constexpr int kLine = 32;   // words between rows' counters
// The largest top_k that goes by slabs, in one workgroup (64 rows of 128256: 40
// 30 us, 37 by bins; a batch with rows of 200 65 against 58), the slabs it sorts,
// and the largest whose rows need no masses of bins.
constexpr int kSlabTopK = 64, kSlabsMax = 1024, kListTopK = 2048;

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

// Lane operations along a wave by DPP: 1, 2, 4 and 8 lanes up within a row of 16,
// then the last lanes of rows 0, 2 and of row 1 to the rows behind them.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t v, uint32_t other) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)other, (int)v, CTRL, ROWS, 0xF, false);
}
#define GOLLEK_ALONG(STEP) \
    STEP(0x111, 0xF) STEP(0x112, 0xF) STEP(0x114, 0xF) STEP(0x118, 0xF) STEP(0x142, 0xA) STEP(0x143, 0xC)
// Inclusive sums up to each lane.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
#define GOLLEK_STEP(C, R) v += dpp<C, R>(v, 0u);
    GOLLEK_ALONG(GOLLEK_STEP)
#undef GOLLEK_STEP
    return v;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {
#define GOLLEK_STEP(C, R) v += ((u64)dpp<C, R>((uint32_t)(v >> 32), 0u) << 32) | dpp<C, R>((uint32_t)v, 0u);
    GOLLEK_ALONG(GOLLEK_STEP)
#undef GOLLEK_STEP
    return v;
}
// The largest of the wave's values, in lane 63.
__device__ __forceinline__ float wave_top(float v) {
#define GOLLEK_STEP(C, R) v = fmaxf(v, __uint_as_float(dpp<C, R>(__float_as_uint(v), 0xFF800000u)));
    GOLLEK_ALONG(GOLLEK_STEP)
#undef GOLLEK_STEP
    return v;
}
#undef GOLLEK_ALONG
template <class V>
__device__ __forceinline__ V last_lane(V v) {
    if constexpr (sizeof(V) == 8) {
        const u64 b = __builtin_bit_cast(u64, v);
        return __builtin_bit_cast(V, ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), 63) << 32) |
                                         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63));
    } else {
        return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
    }
}

// The sum over the workgroup, in every thread.
template <class V>
__device__ V block_sum(V v, RowLds &s) {
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) s.part[threadIdx.x >> 6] = (u64)v;
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
    if (r >= ties) return Border{prefix, prefix == in.key ? in.index : 0x7FFFFFFF};  // (all within `in`)
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

// A row by one workgroup, whatever it holds.
__device__ __forceinline__ void whole_row(const SampleArgs &a, int row, const Wish &wish, float m, RowLds &s) {
    const int tid = (int)threadIdx.x;
    const int64_t base = (int64_t)row * a.stride;
    const Scale sc(m, wish.inv_t, a.shift);

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
        u64 cum = wave_scan(f);
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

// ---- the four launches --------------------------------------------------------

struct Bins {
    float m, inv;
    bool far;
    __device__ __forceinline__ int of(float l) const {
        return l == m || inv == 0.0f ? 0 : (int)fminf((m - l) * inv, (float)(kBins - 1));  // (m infinite: the last)
    }
};
struct Plan {
    int mode;          // see kNone ..
    int from, last;    // bins that are collected (none: 0, -1)
    int bin;           // the border's bin, kBins: none
    uint32_t before;   // tokens in the bins above the border's
    uint32_t tokens;   // of the row that top_k leaves
    float top;         // the row's largest logit
    Bins bins;
    u64 before_mass;   // mass in the bins above the border's
    double target;     // mass that top_p wants (0: its share of the collected tokens' first top_k)
};
enum : int {
    kNone,    // no token
    kWhole,   // the last workgroup alone
    kFree,    // no border with weight below it: every token, by chunks
    kBorder,  // the collected tokens are the border's bin
    kAll,     // every token that may be kept is collected
    kSlabs,   // the same, by the last workgroup itself, from the slabs that top_k reaches
};

struct SampleWs {
    float *tops;          // [rows][chunks * 16] slabs' largest logits
    float *least;         // [rows][chunks * 4] least finite logits
    u64 *mass;            // [rows][parts][kBins]
    u64 *chunk_mass;      // [rows][chunks]
    u64 *list;            // [rows][kList]
    Plan *plan;           // [rows]
    uint32_t *count;      // [rows][parts][kBins]
    uint32_t *chunk_kept; // [rows][chunks]
    uint32_t *listed;     // [rows] kLine apart: rows' counters share no cache line
    int chunks, parts;
    // chunks of a part
    __device__ __forceinline__ int first(int part) const { return (int)((int64_t)part * chunks / parts); }
};

// Logits i .. i + 3 of a row, -inf behind the vocabulary.
__device__ __forceinline__ void load4(const SampleArgs &a, int64_t base, int i, float (&l)[4]) {
    if (a.vec4 && i + 4 <= a.vocab) {
        if (a.type == kF32) {
            const float4 v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.logits) + base + i);
            l[0] = v.x, l[1] = v.y, l[2] = v.z, l[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.logits) + base + i);
            const uint32_t h[4] = {v.x & 0xFFFFu, v.x >> 16, v.y & 0xFFFFu, v.y >> 16};
#pragma unroll
            for (int j = 0; j < 4; j++)
                l[j] = a.type == kBF16 ? __uint_as_float(h[j] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) l[j] = i + j < a.vocab ? load_element(a.logits, a.type, base + i + j) : -__builtin_inff();
    }
}
// A thread's tokens of a chunk: the slabs are waves' quarters of 1024.
__device__ __forceinline__ void load_chunk(const SampleArgs &a, int64_t base, int c, float (&l)[4][4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) load4(a, base, c * kChunk + j * 1024 + 4 * (int)threadIdx.x, l[j]);
}

__global__ __launch_bounds__(kScan) void sample_range_kernel(SampleArgs a, SampleWs ws) {
    const int row = (int)blockIdx.y, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t base = (int64_t)row * a.stride;
    if (blockIdx.x == 0 && tid == 0) ws.listed[kLine * row] = 0;
    for (int c = ws.first((int)blockIdx.x); c < ws.first((int)blockIdx.x + 1); c++) {
        float l[4][4];
        load_chunk(a, base, c, l);
        const int64_t at = (int64_t)row * ws.chunks + c;
        float low = -__builtin_inff();  // the largest of the negated tokens
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float top = wave_top(fmaxf(fmaxf(l[j][0], l[j][1]), fmaxf(l[j][2], l[j][3])));
            if (lane == 63) ws.tops[kChunkSlabs * at + 4 * j + wave] = top;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (l[j][i] > -__builtin_inff()) low = fmaxf(low, -l[j][i]);
        }
        low = wave_top(low);
        if (lane == 63) ws.least[4 * at + wave] = -low;
    }
}

struct Range {
    float top, least;
    int slabs;  // that hold a token
};
// The row's largest and least logit, for a workgroup of THREADS.
template <int THREADS>
__device__ __forceinline__ Range row_range(const SampleWs &ws, int row) {
    __shared__ Range part[THREADS / 64];
    Range r = {-__builtin_inff(), __builtin_inff(), 0};
    for (int i = (int)threadIdx.x; i < kChunkSlabs * ws.chunks; i += THREADS) {
        const float t = ws.tops[(int64_t)row * kChunkSlabs * ws.chunks + i];
        r.top = fmaxf(r.top, t);
        r.slabs += t > -__builtin_inff() ? 1 : 0;
    }
    for (int i = (int)threadIdx.x; i < 4 * ws.chunks; i += THREADS)
        r.least = fminf(r.least, ws.least[(int64_t)row * 4 * ws.chunks + i]);
    r = {wave_top(r.top), -wave_top(-r.least), (int)wave_scan((uint32_t)r.slabs)};
    if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = r;
    __syncthreads();
    r = part[0];
    for (int w = 1; w < THREADS / 64; w++)
        r = {fmaxf(r.top, part[w].top), fminf(r.least, part[w].least), r.slabs + part[w].slabs};
    return r;
}

// Bins of a row: 0 at the largest logit.  far: the last bin is open, and what
// falls into it has weight 0 (below 2^-(S + 1)).
__device__ __forceinline__ Bins row_bins(const SampleArgs &a, const Wish &w, const Range &r) {
    const float reach = (float)((double)(a.shift + 2) * 0.69314718055994531 / w.inv_t);  // (infinite at T = inf)
    const float span = r.top - r.least;                                                  // (or at huge logits)
    const bool far = !(span < reach);
    const float range = far ? reach : span;
    // A range of 0, or of infinity, leaves one bin.
    return {r.top, range > 0.0f ? fminf((float)(kBins - 1) / range, 0x1p100f) : 0.0f, far};
}

// Whether the masses of the bins are needed: not where top_k bounds the list.
__device__ __forceinline__ bool needs_mass(const Wish &w) { return w.has_p && w.top_k > kListTopK; }

// How a row's border is looked for.
enum : int { kEmpty, kNoBorder, kBySlabs, kByBins, kBySearch };
__device__ __forceinline__ int border_way(const SampleArgs &a, const SampleWs &ws, const Wish &w, const Range &r) {
    if (!(r.top > -__builtin_inff())) return kEmpty;
    if (!w.has_p && w.top_k >= a.vocab) return kNoBorder;
    if (w.top_k <= r.slabs && w.top_k <= kSlabTopK && kChunkSlabs * ws.chunks <= kSlabsMax) return kBySlabs;
    // bins do not count tokens of weight 0 that a tiny min_p keeps
    return w.min_p > 0.0 && w.min_p < __builtin_ldexp(1.0, 2 - a.shift) ? kBySearch : kByBins;
}

// Sums over the workgroup of kScan threads, in every thread.
__device__ __forceinline__ void scan_sum(u64 &mass, uint32_t &n, u64 *pm, uint32_t *pn) {
    mass = wave_scan(mass);
    n = wave_scan(n);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) {
        pm[threadIdx.x >> 6] = mass;
        pn[threadIdx.x >> 6] = n;
    }
    __syncthreads();
    mass = 0;
    n = 0;
    for (int w = 0; w < kScan / 64; w++) {
        mass += pm[w];
        n += pn[w];
    }
}

__global__ __launch_bounds__(kScan) void sample_bins_kernel(SampleArgs a, SampleWs ws) {
    __shared__ u64 mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ u64 pm[kScan / 64];
    __shared__ uint32_t pn[kScan / 64];
    const int row = (int)blockIdx.y, part = (int)blockIdx.x, tid = (int)threadIdx.x;
    const int64_t base = (int64_t)row * a.stride;
    const Wish wish = row_wish(a, row);
    // Rows that cannot go by slabs have their first chunk on the way meanwhile.
    const bool early = wish.top_k > kSlabTopK;
    float l[4][4];
    if (early) load_chunk(a, base, ws.first(part), l);
    const Range r = row_range<kScan>(ws, row);
    const int way = border_way(a, ws, wish, r);
    if (way == kBySlabs || way == kBySearch || way == kEmpty) return;  // (nothing to count)
    const Scale sc(r.top, wish.inv_t, a.shift);
    const Bins bins = row_bins(a, wish, r);
    const bool border = way == kByBins, weigh = needs_mass(wish);
    if (border) {
        for (int b = tid; b < kBins; b += kScan) {
            mass[b] = 0;
            count[b] = 0;
        }
        __syncthreads();
    }
    for (int c = ws.first(part); c < ws.first(part + 1); c++) {
        if (!early || c > ws.first(part)) load_chunk(a, base, c, l);
        if (border) {
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const float v = l[j >> 2][j & 3];
                if (!(v > -__builtin_inff())) continue;
                const int b = bins.of(v);
                atomicAdd(&count[b], 1u);  // LDS
                if (weigh && !(bins.far && b == kBins - 1)) atomicAdd(&mass[b], sc.fixed(sc.weight(v)));
            }
        } else {
            u64 t = 0;
            uint32_t n = 0;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const float v = l[j >> 2][j & 3];
                if (!(v > -__builtin_inff())) continue;
                const double w = sc.weight(v);
                if (!(w >= wish.min_p)) continue;
                t += sc.fixed(w);
                n++;
            }
            scan_sum(t, n, pm, pn);
            if (tid == 0) {
                ws.chunk_mass[(int64_t)row * ws.chunks + c] = t;
                ws.chunk_kept[(int64_t)row * ws.chunks + c] = n;
            }
        }
    }
    if (!border) return;
    __syncthreads();
    const int64_t at = ((int64_t)row * ws.parts + part) * kBins;
    for (int b = tid; b < kBins; b += kScan) {
        ws.count[at + b] = count[b];
        if (weigh) ws.mass[at + b] = mass[b];
    }
}

// Adds the tokens of a chunk that bit j of `listed` names (l[j / 4][j % 4]) to
// the row's list; `counts`: a word per wave.
__device__ __forceinline__ void collect(const SampleWs &ws, int row, int c, const float (&l)[4][4], uint32_t listed,
                                        uint32_t *counts, uint32_t *place) {
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t mine = (uint32_t)__builtin_popcount(listed);
    uint32_t upto = wave_scan(mine);  // places: this thread's after those of the threads before
    __syncthreads();
    if (lane == 63) counts[wave] = upto;
    __syncthreads();
    uint32_t sum = 0;
    for (int w = 0; w < kScan / 64; w++) {
        if (w < wave) upto += counts[w];
        sum += counts[w];
    }
    if (sum == 0) return;  // (the same in every thread)
    if (tid == 0) *place = atomicAdd(ws.listed + kLine * row, sum);
    __syncthreads();
    uint32_t p = *place + upto - mine;
#pragma unroll
    for (int j = 0; j < 16; j++) {
        if ((listed >> j) & 1u) {
            if (p < (uint32_t)kList)  // (more: the last launch sees it by the count)
                ws.list[(int64_t)row * kList + p] = ((u64)(0xFFFFFFFFu - logit_key(l[j >> 2][j & 3])) << 32) |
                                                    (uint32_t)(c * kChunk + (j >> 2) * 1024 + 4 * tid + (j & 3));
            p++;
        }
    }
}

// A row's plan, by a workgroup of kScan threads (the same in every thread).
__device__ __forceinline__ Plan make_plan(const SampleArgs &a, const SampleWs &ws, int row) {
    __shared__ u64 cm[kScan / 64];
    __shared__ uint32_t cn[kScan / 64];
    __shared__ int cut_k, cut_p;
    __shared__ uint32_t before_k, in_k, before_p, in_p;
    __shared__ u64 before_mass;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Wish wish = row_wish(a, row);
    const Range r = row_range<kScan>(ws, row);
    const int way = border_way(a, ws, wish, r);
    Plan plan = {kFree, 0, -1, kBins, 0, 0x7FFFFFFF, r.top, row_bins(a, wish, r), 0, 0.0};
    if (way == kEmpty || way == kBySearch || way == kNoBorder) {
        plan.mode = way == kEmpty ? kNone : way == kBySearch ? kWhole : kFree;
        return plan;
    }
    if (way == kBySlabs) {
        plan.mode = kSlabs;
        plan.tokens = (uint32_t)wish.top_k;
        return plan;
    }
    // The row's histogram: bins 2 tid, 2 tid + 1, summed over the parts, and its scan.
    uint2 n = {0, 0};
    u64 w0 = 0, w1 = 0;
    const int64_t at = (int64_t)row * ws.parts * kBins + 2 * tid;
#pragma unroll 16
    for (int p = 0; p < ws.parts; p++) {
        const uint2 v = *reinterpret_cast<const uint2 *>(ws.count + at + p * kBins);
        n.x += v.x;
        n.y += v.y;
    }
    if (needs_mass(wish)) {
#pragma unroll 16
        for (int p = 0; p < ws.parts; p++) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(ws.mass + at + p * kBins);
            w0 += v.x;
            w1 += v.y;
        }
    }
    uint32_t cum = wave_scan(n.x + n.y);  // inclusive
    u64 cmass = wave_scan(w0 + w1);
    if (lane == 63) {
        cn[wave] = cum;
        cm[wave] = cmass;
    }
    if (tid == 0) {
        cut_k = cut_p = kBins;
        in_k = in_p = before_k = before_p = 0;
        before_mass = 0;
    }
    __syncthreads();
    uint32_t all = 0;
    u64 total = 0;
    for (int w = 0; w < kScan / 64; w++) {
        if (w < wave) {
            cum += cn[w];
            cmass += cm[w];
        }
        all += cn[w];
        total += cm[w];
    }
    const double target = wish.top_p * (double)total;  // (of the whole row; used where top_k drops no weight)
    const uint32_t k = (uint32_t)wish.top_k;
    {
        const uint32_t c[3] = {cum - n.x - n.y, cum - n.y, cum};
        const u64 q[3] = {cmass - w0 - w1, cmass - w1, cmass};
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (k < all && c[j] < k && c[j + 1] >= k) {
                cut_k = 2 * tid + j;
                before_k = c[j];
                in_k = c[j + 1] - c[j];
            }
            if (needs_mass(wish) && (double)q[j] < target && !((double)q[j + 1] < target)) {
                cut_p = 2 * tid + j;
                before_p = c[j];
                in_p = c[j + 1] - c[j];
                before_mass = q[j];
            }
        }
    }
    __syncthreads();
    const bool k_cuts = cut_k < kBins && !(plan.bins.far && cut_k == kBins - 1);  // drops weight
    plan.tokens = k < all ? k : all;
    if (k_cuts && before_k + in_k <= (uint32_t)kList) {
        plan.mode = kAll;
        plan.last = cut_k;
    } else if (wish.has_p && !needs_mass(wish) && !k_cuts) {
        // fewer tokens than top_k, all of them or all that have weight
        plan.mode = kAll;
        plan.last = cut_k < kBins ? cut_k - 1 : kBins - 1;
        plan.tokens = cut_k < kBins ? before_k : all;
    } else if (k_cuts) {
        plan.mode = wish.has_p || in_k > (uint32_t)kList ? kWhole : kBorder;
        plan.bin = plan.from = plan.last = cut_k;
        plan.before = before_k;
    } else if (wish.has_p && before_p + in_p <= (uint32_t)kList) {
        plan.mode = kAll;
        plan.last = cut_p;
        plan.tokens = before_p + in_p;
        plan.target = target;
    } else if (wish.has_p) {
        plan.mode = in_p > (uint32_t)kList ? kWhole : kBorder;
        plan.bin = plan.from = plan.last = cut_p;
        plan.before = before_p;
        plan.before_mass = before_mass;
        plan.target = target;
    }
    return plan;
}

__global__ __launch_bounds__(kScan) void sample_plan_kernel(SampleArgs a, SampleWs ws) {
    const int row = (int)blockIdx.x;
    const Plan plan = make_plan(a, ws, row);
    if (threadIdx.x == 0) ws.plan[row] = plan;
}

// PLAN: every workgroup makes its row's plan (part 0 leaves it for the last launch).
template <bool PLAN>
__global__ __launch_bounds__(kScan) void sample_collect_kernel(SampleArgs a, SampleWs ws) {
    __shared__ u64 pm[kScan / 64];
    __shared__ uint32_t pn[kScan / 64], cn[kScan / 64];
    __shared__ uint32_t place;
    const int row = (int)blockIdx.y, part = (int)blockIdx.x, tid = (int)threadIdx.x, wave = tid >> 6;
    const int64_t base = (int64_t)row * a.stride;
    Plan plan;
    if constexpr (PLAN) {
        plan = make_plan(a, ws, row);
        if (part == 0 && tid == 0) ws.plan[row] = plan;
    } else {
        plan = ws.plan[row];
    }
    const Wish wish = row_wish(a, row);
    if (plan.mode == kNone || plan.mode == kWhole || plan.mode == kSlabs) return;
    if (plan.mode == kFree && !wish.has_p && wish.top_k >= a.vocab) return;  // (the second launch has its masses)
    const Scale sc(plan.top, wish.inv_t, a.shift);
    const float *const tops = ws.tops + (int64_t)row * kChunkSlabs * ws.chunks;
    // The bins of tokens that are collected, or whose mass counts.
    const int deepest = plan.mode == kAll || plan.last > plan.bin - 1 ? plan.last : plan.bin - 1;
    auto concerns = [&](float top) { return top > -__builtin_inff() && plan.bins.of(top) <= deepest; };
    for (int c = ws.first(part); c < ws.first(part + 1); c++) {
        bool any = plan.mode != kAll;  // (then the chunk's mass is written, if it is 0)
#pragma unroll
        for (int j = 0; j < kChunkSlabs; j++) any |= concerns(tops[kChunkSlabs * c + j]);
        if (!any) continue;
        float l[4][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (concerns(tops[kChunkSlabs * c + 4 * j + wave])) {
                load4(a, base, c * kChunk + j * 1024 + 4 * tid, l[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) l[j][i] = -__builtin_inff();
            }
        }
        uint32_t listed = 0;  // bit j: token j is collected
        u64 t = 0;
        uint32_t kept = 0;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const float v = l[j >> 2][j & 3];
            if (!(v > -__builtin_inff())) continue;
            const int b = plan.bins.of(v);
            if (b >= plan.from && b <= plan.last) {
                listed |= 1u << j;
            } else if (plan.mode != kAll && b < plan.bin) {
                const double w = sc.weight(v);
                if (w >= wish.min_p) {
                    t += sc.fixed(w);
                    kept++;
                }
            }
        }
        if (plan.mode != kAll) {
            scan_sum(t, kept, pm, pn);
            if (tid == 0) {
                ws.chunk_mass[(int64_t)row * ws.chunks + c] = t;
                ws.chunk_kept[(int64_t)row * ws.chunks + c] = kept;
            }
        }
        collect(ws, row, c, l, listed, cn, &place);
    }
}

// Inclusive scan of a value per thread over the workgroup; `total` its end.
__device__ __forceinline__ u64 block_scan(u64 v, u64 &total, RowLds &s) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) s.part[wave] = v;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kWaves; w++) {
        if (w < wave) v += s.part[w];
        total += s.part[w];
    }
    return v;
}

struct SortLds {
    u64 list[kList], spare[kList];
    uint32_t slot[kThreads];
    uint32_t most;
    float span[2 * kWaves];
};

// Sorts the first n (up to kList) of s.list, whose values differ, upwards.
// bucket(v): a number in [0, kThreads) that does not fall as v rises.  Every
// value goes to its bucket and finds its place there by counting the smaller
// ones; with more than 128 values in a bucket (equal logits side by side) a bitonic sort.
template <class BUCKET>
__device__ void sort_list(SortLds &s, RowLds &rl, int n, BUCKET &&bucket) {
    const int tid = (int)threadIdx.x;
    if (n <= 64) {
        if (tid < 64) {
            const u64 v = tid < n ? s.list[tid] : 0;
            int below = 0;
            for (int j = 0; j < n; j++) below += s.list[j] < v ? 1 : 0;
            __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses complete in order)
            if (tid < n) s.list[below] = v;
        }
        __syncthreads();
        return;
    }
    s.slot[tid] = 0;
    if (tid == 0) s.most = 0;
    __syncthreads();
    constexpr int kPer = kList / kThreads;
    u64 v[kPer];
    int b[kPer];
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const int i = tid + j * kThreads;
        v[j] = i < n ? s.list[i] : 0;
        b[j] = i < n ? bucket(v[j]) : 0;
        if (i < n) atomicAdd(&s.slot[b[j]], 1u);  // LDS
    }
    __syncthreads();
    const uint32_t mine = s.slot[tid];
    uint32_t most = mine;
    for (int d = 1; d < 64; d <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d));
    if ((tid & 63) == 0) atomicMax(&s.most, most);  // LDS
    u64 total;
    const uint32_t end = (uint32_t)block_scan(mine, total, rl);
    if (s.most <= 128) {  // (block_scan's barriers stand between)
        __syncthreads();
        s.slot[tid] = end - mine;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; j++)
            if (tid + j * kThreads < n) s.spare[atomicAdd(&s.slot[b[j]], 1u)] = v[j];
        __syncthreads();
        // s.slot[b] is the bucket's end now, s.slot[b - 1] its start
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            if (tid + j * kThreads >= n) continue;
            const uint32_t from = b[j] > 0 ? s.slot[b[j] - 1] : 0u, to = s.slot[b[j]];
            uint32_t place = from;
            for (uint32_t i = from; i < to; i += 4) {  // (four reads on the way at a time)
#pragma unroll
                for (uint32_t q = 0; q < 4; q++) place += s.spare[i + q < to ? i + q : i] < v[j] && i + q < to ? 1u : 0u;
            }
            s.list[place] = v[j];
        }
        __syncthreads();
        return;
    }
    int size = 128;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += kThreads) s.list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = tid; t < size / 2; t += kThreads) {
                const int i = 2 * t - (t & (j - 1)), o = i + j;
                const u64 x = s.list[i], y = s.list[o];
                if ((x > y) == ((i & k) == 0)) {
                    s.list[i] = y;
                    s.list[o] = x;
                }
            }
            __syncthreads();
        }
}

// The tokens of a row that a top_k of k can keep, into the list (its length is
// returned; past kList only counted): k slabs at least hold a token as large as
// the k-th largest slab maximum, so none below it is among the first k.  Of that
// maximum's key the upper half suffices, found by a histogram of the first byte,
// then of the second.
__device__ __forceinline__ int collect_slabs(const SampleArgs &a, const SampleWs &ws, int row, uint32_t k, SortLds &so,
                                             RowLds &s) {
    static_assert(kSlabsMax <= kThreads, "a thread a slab");
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, slabs = kChunkSlabs * ws.chunks;
    const uint32_t key = tid < slabs ? logit_key(ws.tops[(int64_t)row * slabs + tid]) : 0u;
    uint32_t floor = 0;
#pragma unroll
    for (int at = 24; at >= 16; at -= 8) {
        if (tid < 256) s.count[tid] = 0;
        if (tid == 0) so.most = s.found = 0;
        __syncthreads();
        if (key > 0 && (at == 24 || key >> 24 == floor >> 24)) atomicAdd(&s.count[(key >> at) & 255u], 1u);  // LDS
        __syncthreads();
        const uint32_t mine = tid < 256 ? s.count[255 - tid] : 0u;  // from the top
        uint32_t end = wave_scan(mine);
        if (lane == 63) s.part[wave] = end;
        __syncthreads();
        for (int w = 0; w < wave; w++) end += (uint32_t)s.part[w];
        if (end >= k && end - mine < k) {  // one thread
            s.digit = (uint32_t)(255 - tid);
            s.before_count = end - mine;
        }
        __syncthreads();
        floor |= s.digit << at;
        k -= s.before_count;
    }
    if (floor == 0) floor = 1;  // (0 is no token)
    if (key >= floor) so.slot[atomicAdd(&s.found, 1)] = (uint32_t)tid;  // LDS
    __syncthreads();
    const int n = s.found;
    const int64_t base = (int64_t)row * a.stride;
    constexpr int kAhead = 4;
    for (int i0 = wave; i0 < n; i0 += kAhead * kWaves) {
        float l[kAhead][4];
        int at[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int i = i0 + j * kWaves;
            at[j] = i < n ? 256 * (int)so.slot[i] + 4 * lane : a.vocab;  // (a slab is 256 neighbours)
            load4(a, base, at[j], l[j]);
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            uint32_t count = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) count += logit_key(l[j][i]) >= floor ? 1u : 0u;
            const uint32_t upto = wave_scan(count);
            uint32_t place = 0;
            if (lane == 63 && upto > 0) place = atomicAdd(&so.most, upto);  // LDS
            place = (uint32_t)__builtin_amdgcn_readlane((int)place, 63) + upto - count;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t t = logit_key(l[j][i]);
                if (t < floor) continue;
                if (place < (uint32_t)kList) so.list[place] = ((u64)(0xFFFFFFFFu - t) << 32) | (uint32_t)(at[j] + i);
                place++;
            }
        }
    }
    __syncthreads();
    return (int)so.most;
}

__device__ __forceinline__ void write_token(const SampleArgs &a, int row, int token, double w, u64 total, uint32_t kept) {
    a.tokens[row] = token;
    if (a.probs != nullptr) a.probs[row] = (float)(__builtin_ldexp(w, a.shift) / (double)total);
    if (a.kept != nullptr) a.kept[row] = (int32_t)kept;
}
__device__ __forceinline__ void write_none(const SampleArgs &a, int row) {
    a.tokens[row] = -1;
    if (a.probs != nullptr) a.probs[row] = 0.0f;
    if (a.kept != nullptr) a.kept[row] = 0;
}
// A collected token: upper half the inverted key, lower half the index.
__device__ __forceinline__ u64 entry_of(uint32_t key, int index) { return ((u64)(0xFFFFFFFFu - key) << 32) | (uint32_t)index; }
__device__ __forceinline__ float logit_of(u64 entry) { return key_logit(0xFFFFFFFFu - (uint32_t)(entry >> 32)); }

// The draw from up to 128 collected tokens, which hold every one that may be
// kept: two a lane of one wave, without a barrier, their places by counting, by
// key and then by index.  tokens: what top_k leaves; target: the mass that top_p
// wants, 0: its share of theirs.
__device__ void draw_few(const SampleArgs &a, int row, const Wish &wish, const Scale &sc, SortLds &so, int n,
                         uint32_t tokens, double target) {
    const int tid = (int)threadIdx.x;
    u64 v[2] = {~0ull, ~0ull};
#pragma unroll
    for (int j = 0; j < 2; j++) {
        if (tid + 64 * j < n) v[j] = so.list[tid + 64 * j];
    }
    auto place = [&](int count, bool (&in)[2]) {  // those of `in` below each value, of the first `count`
        __builtin_amdgcn_wave_barrier();          // (a wave's LDS accesses complete in order)
        int below[2] = {0, 0};
        for (int i = 0; i < count; i++) {
            const u64 o = so.list[i];
            below[0] += o < v[0] ? 1 : 0;
            below[1] += o < v[1] ? 1 : 0;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < 2; j++)
            if (in[j]) so.list[below[j]] = v[j];
        __builtin_amdgcn_wave_barrier();
    };
    // Inclusive sums along 2 lane, 2 lane + 1, and the whole.
    auto sums = [&](const u64 (&f)[2], u64 (&upto)[2]) {
        const u64 t = wave_scan(f[0] + f[1]);
        upto[0] = t - f[1];
        upto[1] = t;
        return last_lane(t);
    };
    bool in[2] = {tid < n, tid + 64 < n};
    place(n, in);
    const int k = tokens < (uint32_t)n ? (int)tokens : n;
    double w[2];
    u64 f[2], upto[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int i = 2 * tid + j;
        v[j] = so.list[i];
        in[j] = i < k;
        w[j] = in[j] ? sc.weight(logit_of(v[j])) : 0.0;
        f[j] = in[j] ? sc.fixed(w[j]) : 0;
    }
    u64 total = sums(f, upto);
    const double border = target > 0.0 ? target : wish.top_p * (double)total;
    int kept = 0;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        in[j] = in[j] && (!wish.has_p || (double)(upto[j] - f[j]) < border) && w[j] >= wish.min_p;
        kept += __builtin_popcountll(__ballot(in[j]));
    }
    // by index: the kept ones are the first `kept` of the order
#pragma unroll
    for (int j = 0; j < 2; j++) {
        v[j] = (v[j] << 32) | (0xFFFFFFFFu - (uint32_t)(v[j] >> 32));
        so.list[2 * tid + j] = v[j];
    }
    place(kept, in);
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int i = 2 * tid + j;
        v[j] = so.list[i];
        w[j] = i < kept ? sc.weight(key_logit((uint32_t)v[j])) : 0.0;
        f[j] = i < kept ? sc.fixed(w[j]) : 0;
    }
    total = sums(f, upto);
    const double point = wish.u * (double)total;
#pragma unroll
    for (int j = 0; j < 2; j++)
        if (f[j] > 0 && (double)upto[j] > point && !((double)(upto[j] - f[j]) > point))  // one lane, once
            write_token(a, row, (int)(v[j] >> 32), w[j], total, (uint32_t)kept);
}

// The first n of so.list in order.
__device__ __forceinline__ void sort_by_logit(const SampleArgs &a, SortLds &so, RowLds &s, int n) {
    const int tid = (int)threadIdx.x;
    float low = __builtin_inff(), high = -__builtin_inff();
    for (int i = tid; i < n; i += kThreads) {
        low = fminf(low, logit_of(so.list[i]));
        high = fmaxf(high, logit_of(so.list[i]));
    }
    low = -wave_top(-low);
    high = wave_top(high);
    if ((tid & 63) == 63) {
        so.span[tid >> 6] = low;
        so.span[kWaves + (tid >> 6)] = high;
    }
    __syncthreads();
    low = __builtin_inff();
    high = -__builtin_inff();
    for (int w = 0; w < kWaves; w++) {
        low = fminf(low, so.span[w]);
        high = fmaxf(high, so.span[kWaves + w]);
    }
    // Few keys (16-bit logits have the lower bits of theirs all alike): the buckets
    // are shared out among them, and a key's go by index.  (4 rows of 151936 bf16,
    // top_p 0.95: 49 us, 57 where such crowds were sorted bitonically.)
    const uint32_t first = 0xFFFFFFFFu - logit_key(high);
    const int zeros = low == high ? 31 : a.type == kBF16 ? 16 : a.type == kF16 ? 13 : 0;
    const uint32_t keys = ((0xFFFFFFFFu - logit_key(low) - first) >> zeros) + 1u;
    if (keys <= (uint32_t)kThreads / 2) {
        const uint32_t each = (uint32_t)kThreads / keys;
        const float share = (float)each / (float)a.vocab;
        sort_list(so, s, n, [&](u64 v) {
            const uint32_t at = (uint32_t)((float)(uint32_t)v * share);
            return (int)((((uint32_t)(v >> 32) - first) >> zeros) * each + min(at, each - 1));
        });
        return;
    }
    const float wide = high - low;  // (infinite or 0: one bucket)
    const float inv = wide > 0.0f && wide < 0x1p126f ? fminf(1.0f / wide, 0x1p100f) : 0.0f;
    sort_list(so, s, n, [&](u64 v) {  // (finer at the lower end, where tokens are denser)
        const float x = inv > 0.0f ? fminf((high - logit_of(v)) * inv, 1.0f) : 0.0f;
        return (int)(x * (0.4f + 0.6f * x) * (float)(kThreads - 1));
    });
}

// One workgroup per row.
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleArgs a, SampleWs ws) {
    __shared__ RowLds s;
    __shared__ SortLds so;
    __shared__ u64 chunk[kThreads];
    __shared__ int which;
    __shared__ u64 before_chunk;
    __shared__ uint32_t in_chunk;
    constexpr int kPer = kList / kThreads;
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x;
    const int64_t base = (int64_t)row * a.stride;
    const Wish wish = row_wish(a, row);
    const Plan plan = ws.plan[row];
    if (plan.mode == kNone) {
        if (tid == 0) write_none(a, row);
        return;
    }
    const bool all = plan.mode == kAll || plan.mode == kSlabs;  // every token that may be kept is in the list
    int n = 0;
    if (plan.mode == kSlabs) {
        n = collect_slabs(a, ws, row, plan.tokens, so, s);
    } else if (plan.mode == kAll || plan.mode == kBorder) {
        n = (int)ws.listed[kLine * row];
        for (int i = tid; i < n && i < kList; i += kThreads) so.list[i] = ws.list[(int64_t)row * kList + i];
        __syncthreads();
    }
    if (plan.mode == kWhole || n > kList) {
        whole_row(a, row, wish, plan.top, s);
        return;
    }
    const Scale sc(plan.top, wish.inv_t, a.shift);
    if (all && n <= 128) {
        if (tid < 64) draw_few(a, row, wish, sc, so, n, plan.tokens, plan.target);
        return;
    }

    // The collected tokens in order (upper half the inverted key, lower half the
    // index), their weights, and the border among them.
    Border border = {0, 0x7FFFFFFF};
    uint32_t kept = 0;
    u64 f[kPer];
    bool keep[kPer];
    chunk[tid] = 0;
    if (n > 0) {
        sort_by_logit(a, so, s, n);
        const int k = all && plan.tokens < (uint32_t)n ? (int)plan.tokens : n;
        u64 sum = 0, total;
        double w[kPer];
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const int i = kPer * tid + j;
            w[j] = i < k ? sc.weight(logit_of(so.list[i])) : 0.0;
            f[j] = i < k ? sc.fixed(w[j]) : 0;
            sum += f[j];
        }
        u64 before = plan.before_mass + block_scan(sum, total, s) - sum;
        const double target = plan.target > 0.0 ? plan.target : wish.top_p * (double)total;
        uint32_t in = 0;
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const int i = kPer * tid + j;
            // (kBorder without a target: top_k's border)
            const bool inside = i < k && (plan.mode == kBorder && !(plan.target > 0.0) ? plan.before + (uint32_t)i < plan.tokens
                                                                                       : !wish.has_p || (double)before < target);
            before += f[j];
            in += inside ? 1u : 0u;
            keep[j] = inside && w[j] >= wish.min_p;
            if (!keep[j]) continue;
            kept++;
            if (f[j] > 0) atomicAdd(&chunk[(uint32_t)so.list[i] / kChunk], f[j]);  // LDS
        }
        if (plan.mode == kBorder) {
            in = block_sum(in, s);
            border = {0xFFFFFFFFu - (uint32_t)(so.list[in - 1] >> 32), (int)(uint32_t)so.list[in - 1]};
        }
    }
    __syncthreads();
    // The chunks' kept mass, and the one that the random number falls into.
    u64 mine = tid < ws.chunks ? chunk[tid] : 0;
    if (!all && tid < ws.chunks) {
        mine += ws.chunk_mass[(int64_t)row * ws.chunks + tid];
        kept += ws.chunk_kept[(int64_t)row * ws.chunks + tid];
    }
    kept = block_sum(kept, s);
    if (plan.mode == kFree && wish.min_p == 0.0 && plan.tokens < kept) kept = plan.tokens;  // top_k drops weights of 0
    u64 total;
    const u64 upto = block_scan(mine, total, s);
    const double point = wish.u * (double)total;
    if (tid == 0) in_chunk = 0;
    if (mine > 0 && !((double)(upto - mine) > point) && (double)upto > point) {  // one thread
        which = tid;
        before_chunk = upto - mine;
    }
    __syncthreads();
    u64 cum = before_chunk;
    if (all) {
        // the chunk's kept tokens by index: upper half the index, lower half the key
        u64 v[kPer];
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const int i = kPer * tid + j;
            v[j] = i < n ? so.list[i] : 0;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; j++)
            if (kPer * tid + j < n && keep[j] && (int)((uint32_t)v[j] / kChunk) == which)
                so.list[atomicAdd(&in_chunk, 1u)] = (v[j] << 32) | (0xFFFFFFFFu - (uint32_t)(v[j] >> 32));  // LDS
        __syncthreads();
        const int m = (int)in_chunk;
        sort_list(so, s, m, [](u64 e) { return (int)((uint32_t)(e >> 32) % kChunk / (kChunk / kThreads)); });
        u64 sum = 0, end;
        double w[kPer];
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const int i = kPer * tid + j;
            w[j] = i < m ? sc.weight(key_logit((uint32_t)so.list[i])) : 0.0;
            f[j] = i < m ? sc.fixed(w[j]) : 0;
            sum += f[j];
        }
        cum += block_scan(sum, end, s) - sum;
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            if (f[j] > 0 && !((double)cum > point) && (double)(cum + f[j]) > point)  // one thread, once
                write_token(a, row, (int)(so.list[kPer * tid + j] >> 32), w[j], total, kept);
            cum += f[j];
        }
        return;
    }
    const int i0 = which * kChunk + 4 * tid;
    float l[4];
    load4(a, base, i0, l);
    double w[4];
    u64 sum = 0, end;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t key = logit_key(l[j]);
        f[j] = 0;
        w[j] = 0.0;
        if (key != 0 && border.keeps(key, i0 + j)) {
            w[j] = sc.weight(l[j]);
            if (w[j] >= wish.min_p) f[j] = sc.fixed(w[j]);
        }
        sum += f[j];
    }
    cum += block_scan(sum, end, s) - sum;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (f[j] > 0 && !((double)cum > point) && (double)(cum + f[j]) > point) write_token(a, row, i0 + j, w[j], total, kept);
        cum += f[j];
    }
}

// ---- vocabularies that a workgroup holds ------------------------------------------

// A row of up to PER * 1024 logits in the registers of one workgroup: thread t's
// are 4 t .. 4 t + 3 of every 4096, so everything else is one launch (16 rows of
// 8000: top_k 40 7.8 us, four launches 23.0; top_p 0.9 17.1 against 23.7; no filter
// 9.6 against 18.3).  The same borders: a small top_k by the largest of slabs (of 32
// or 64 tokens here), others by a histogram, top_k's first, then top_p's among what
// that leaves, each exact by sorting its bin.
template <int PER>
__global__ __launch_bounds__(kThreads) void sample_small_kernel(SampleArgs a) {
    __shared__ RowLds s;
    __shared__ SortLds so;
    __shared__ u64 mass[kBins];
    __shared__ uint32_t count[kBins];
    constexpr int kGroup = PER <= 8 ? 8 : 16, kSlabs = PER / 4 * kThreads / kGroup;  // lanes of a slab
    __shared__ float tops[kSlabs], least_part[kWaves];
    __shared__ uint32_t floor_key;
    __shared__ u64 sums[PER / 4][kWaves];
    __shared__ int cut;
    __shared__ uint32_t before, inside;
    __shared__ u64 before_mass;
    constexpr int kChunks = PER / 4, kPer = kList / kThreads;
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t base = (int64_t)row * a.stride;
    float l[kChunks][4];
#pragma unroll
    for (int c = 0; c < kChunks; c++) load4(a, base, c * kChunk + 4 * tid, l[c]);
    const Wish wish = row_wish(a, row);
    auto index = [&](int c, int i) { return c * kChunk + 4 * tid + i; };

    float low = -__builtin_inff();  // the largest of the negated tokens
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
        float t = fmaxf(fmaxf(l[c][0], l[c][1]), fmaxf(l[c][2], l[c][3]));
        auto up = [&](uint32_t v) { t = fmaxf(t, __uint_as_float(v)); };
        up(dpp<0x111, 0xF>(__float_as_uint(t), 0xFF800000u));  // (as wave_top, within the group)
        up(dpp<0x112, 0xF>(__float_as_uint(t), 0xFF800000u));
        up(dpp<0x114, 0xF>(__float_as_uint(t), 0xFF800000u));
        if constexpr (kGroup == 16) up(dpp<0x118, 0xF>(__float_as_uint(t), 0xFF800000u));
        if (tid % kGroup == kGroup - 1) tops[(c * kThreads + tid) / kGroup] = t;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (l[c][i] > -__builtin_inff()) low = fmaxf(low, -l[c][i]);
    }
    low = wave_top(low);
    if (lane == 63) least_part[wave] = -low;
    if (tid < kBins) count[tid] = 0;
    if (tid == 0) so.most = 0;
    __syncthreads();
    Range r = {-__builtin_inff(), __builtin_inff(), 0};
    {
        // every wave reads all of them
        for (int i = lane; i < kSlabs; i += 64) {
            r.top = fmaxf(r.top, tops[i]);
            r.slabs += tops[i] > -__builtin_inff() ? 1 : 0;
        }
        r = {last_lane(wave_top(r.top)), lane < kWaves ? least_part[lane] : __builtin_inff(),
             (int)last_lane(wave_scan((uint32_t)r.slabs))};
        r.least = -last_lane(wave_top(-r.least));
    }
    if (!(r.top > -__builtin_inff())) {
        if (tid == 0) write_none(a, row);
        return;
    }
    const Scale sc(r.top, wish.inv_t, a.shift);
    const bool filtered = wish.has_p || wish.top_k < a.vocab;
    // (bins do not count tokens of weight 0)
    bool whole = filtered && wish.min_p > 0.0 && wish.min_p < __builtin_ldexp(1.0, 2 - a.shift);

    if (wish.top_k <= kSlabTopK && wish.top_k <= r.slabs) {
        // The top_k-th largest slab maximum, to 16 bits of its key, by one wave.
        if (wave == 0) {
            constexpr int kOwn = kSlabs / 64;
            uint32_t key[kOwn], found = 0;
#pragma unroll
            for (int j = 0; j < kOwn; j++) key[j] = logit_key(tops[lane + 64 * j]);
            for (int bit = 31; bit >= 16; bit--) {
                const uint32_t next = found | (1u << bit);
                int n = 0;
#pragma unroll
                for (int j = 0; j < kOwn; j++) n += __builtin_popcountll(__ballot(key[j] >= next));
                if (n >= wish.top_k) found = next;
            }
            if (lane == 0) floor_key = found;
        }
        __syncthreads();
        uint32_t floor = floor_key;
        if (floor == 0) floor = 1;
#pragma unroll
        for (int c = 0; c < kChunks; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t k = logit_key(l[c][i]);
                if (k < floor) continue;
                const uint32_t place = atomicAdd(&so.most, 1u);  // LDS
                if (place < 128) so.list[place] = entry_of(k, index(c, i));
            }
        __syncthreads();
        const int n = (int)so.most;
        if (n <= 128) {
            if (tid < 64) draw_few(a, row, wish, sc, so, n, (uint32_t)wish.top_k, 0.0);
            return;
        }
    }

    Border border = {0, 0x7FFFFFFF};
    uint32_t limit = 0x7FFFFFFF;  // tokens that top_k leaves
    if (filtered && !whole) {
        const Bins bins = row_bins(a, wish, r);
        // The tokens of bin `cut` within the border, sorted; false: more than the list holds.
        auto sort_bin = [&](uint32_t n) {
            if (n > (uint32_t)kList) return false;
            if (tid == 0) so.most = 0;
            __syncthreads();
#pragma unroll
            for (int c = 0; c < kChunks; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t k = logit_key(l[c][i]);
                    if (k == 0 || bins.of(l[c][i]) != cut || !border.keeps(k, index(c, i))) continue;
                    so.list[atomicAdd(&so.most, 1u)] = entry_of(k, index(c, i));  // LDS
                }
            __syncthreads();
            sort_by_logit(a, so, s, (int)so.most);
            return true;
        };
#pragma unroll
        for (int c = 0; c < kChunks; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (l[c][i] > -__builtin_inff()) atomicAdd(&count[bins.of(l[c][i])], 1u);  // LDS
        if (tid == 0) cut = kBins;
        __syncthreads();
        const uint32_t mine = tid < kBins ? count[tid] : 0u;
        u64 tokens;
        const uint32_t end = (uint32_t)block_scan(mine, tokens, s), k = (uint32_t)wish.top_k;
        if (k < (uint32_t)tokens) {
            limit = k;
            if (end >= k && end - mine < k && mine > 0) {  // one thread
                cut = tid;
                before = end - mine;
                inside = mine;
            }
            __syncthreads();
            if (!(bins.far && cut == kBins - 1)) {  // (there it drops no weight)
                whole = !sort_bin(inside);
                const u64 last = so.list[whole ? 0 : k - before - 1];
                border = {0xFFFFFFFFu - (uint32_t)(last >> 32), (int)(uint32_t)last};
            }
        }
        if (wish.has_p && !whole) {
            __syncthreads();
            if (tid < kBins) {
                mass[tid] = 0;
                count[tid] = 0;
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < kChunks; c++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t key = logit_key(l[c][i]);
                    if (key == 0 || !border.keeps(key, index(c, i))) continue;
                    const int b = bins.of(l[c][i]);
                    if (bins.far && b == kBins - 1) continue;  // (weight 0)
                    atomicAdd(&count[b], 1u);  // LDS
                    atomicAdd(&mass[b], sc.fixed(sc.weight(l[c][i])));
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            __syncthreads();
            const u64 m = tid < kBins ? mass[tid] : 0;
            u64 total;
            const u64 upto = block_scan(m, total, s);
            const double target = wish.top_p * (double)total;
            if (m > 0 && (double)(upto - m) < target && !((double)upto < target)) {  // one thread
                cut = tid;
                inside = count[tid];
                before_mass = upto - m;
            }
            __syncthreads();
            whole = !sort_bin(inside);
            const int n = whole ? 0 : (int)inside;
            u64 f[kPer], sum = 0, all;
#pragma unroll
            for (int j = 0; j < kPer; j++) {
                const int i = kPer * tid + j;
                f[j] = i < n ? sc.fixed(sc.weight(logit_of(so.list[i]))) : 0;
                sum += f[j];
            }
            u64 at = before_mass + block_scan(sum, all, s) - sum;
            uint32_t in = 0;
#pragma unroll
            for (int j = 0; j < kPer; j++) {
                in += kPer * tid + j < n && (double)at < target ? 1u : 0u;
                at += f[j];
            }
            in = block_sum(in, s);
            const u64 last = so.list[in > 0 ? in - 1 : 0];
            border = {0xFFFFFFFFu - (uint32_t)(last >> 32), (int)(uint32_t)last};
        }
    }
    if (whole) {
        whole_row(a, row, wish, r.top, s);
        return;
    }

    // The draw: the kept mass of every chunk and wave, which one holds the point,
    // and the token in it.
    auto weigh = [&](int c, int i, double &w) {
        const uint32_t k = logit_key(l[c][i]);
        w = 0.0;
        if (k == 0 || !border.keeps(k, index(c, i))) return false;
        w = sc.weight(l[c][i]);
        return w >= wish.min_p;
    };
    uint32_t kept = 0;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
        u64 f = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            double w;
            if (!weigh(c, i, w)) continue;
            f += sc.fixed(w);
            kept++;
        }
        f = wave_scan(f);
        if (lane == 63) sums[c][wave] = f;
        __builtin_amdgcn_sched_barrier(0);  // (the weights of all chunks at once have no registers)
    }
    kept = block_sum(kept, s);  // (its barriers stand between)
    if (!wish.has_p && wish.min_p == 0.0 && limit < kept) kept = limit;  // top_k drops weights of 0
    const u64 part = tid < kChunks * kWaves ? sums[tid / kWaves][tid % kWaves] : 0;
    u64 total;
    const u64 upto = block_scan(part, total, s);
    const double point = wish.u * (double)total;
    if (part > 0 && !((double)(upto - part) > point) && (double)upto > point) {  // one thread
        cut = tid;
        before_mass = upto - part;
    }
    __syncthreads();
    if (cut % kWaves != wave) return;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
        if (cut / kWaves != c) continue;
        double w[4];
        u64 f[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[i] = weigh(c, i, w[i]) ? sc.fixed(w[i]) : 0;
            sum += f[i];
        }
        u64 cum = before_mass + wave_scan(sum) - sum;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (f[i] > 0 && !((double)cum > point) && (double)(cum + f[i]) > point)  // one lane, once
                write_token(a, row, index(c, i), w[i], total, kept);
            cum += f[i];
        }
    }
}

// Workgroups a row is dealt to: one a chunk, so that rows whose weights are
// summed do not wait behind others, up to the 64 whose histograms are read back.
constexpr int kDealt = 2048, kMaxParts = 64;
int row_parts(int rows, int chunks) {
    int want = kDealt / rows;
    if (want > kMaxParts) want = kMaxParts;
    if (want > chunks) want = chunks;
    return want > 1 ? want : 1;
}

struct SampleLayout {
    size_t tops, least, mass, chunk_mass, list, plan, count, chunk_kept, listed, total;
    int chunks, parts;
};
SampleLayout sample_layout(int rows, int vocab) {
    SampleLayout o = {};
    o.chunks = (vocab + kChunk - 1) / kChunk;
    o.parts = row_parts(rows > 0 ? rows : 1, o.chunks);
    auto take = [&](size_t bytes) {
        const size_t at = o.total;
        o.total += (bytes + 255) / 256 * 256;
        return at;
    };
    // Histograms: room for those of any smaller batch too (its rows are dealt to
    // more parts: 93 of 128256 to 22, 96 to 21), so that a workspace never shrinks
    // with rows or vocab.
    const int64_t spread = (int64_t)rows * (o.chunks < kMaxParts ? o.chunks : kMaxParts);
    const int64_t dealt = spread < kDealt ? spread : kDealt;
    const size_t r = (size_t)rows, rc = r * o.chunks, rb = (size_t)(dealt > rows ? dealt : rows) * kBins;
    o.tops = take(rc * kChunkSlabs * sizeof(float));
    o.least = take(rc * 4 * sizeof(float));
    o.mass = take(rb * sizeof(u64));
    o.chunk_mass = take(rc * sizeof(u64));
    o.list = take(r * kList * sizeof(u64));
    o.plan = take(r * sizeof(Plan));
    o.count = take(rb * sizeof(uint32_t));
    o.chunk_kept = take(rc * sizeof(uint32_t));
    o.listed = take(r * kLine * sizeof(uint32_t));
    return o;
}

}  // namespace

// The largest vocabulary that goes to one workgroup: past it the weights alone take
// it longer than the launches (16000: no filter 13.5 against 17.3 us, top_p 0.9 23.4
// against 23.0).
constexpr int kSmallVocab = 16384;

size_t sample_workspace_bytes(int rows, int vocab) {
    return vocab <= kSmallVocab ? 0 : sample_layout(rows, vocab).total;
}

hipError_t launch_sample(const void *logits, int logits_type, int rows, int vocab, int64_t stride,
                         const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                         const float *u, int32_t *tokens, float *probs, int32_t *kept, uint8_t *workspace,
                         hipStream_t stream) {
    if (rows <= 0) return hipSuccess;
    int bits = 1;
    while ((1ll << bits) <= vocab) bits++;
    const uintptr_t size = logits_type == kF32 ? 4 : 2;
    const bool vec4 = ((reinterpret_cast<uintptr_t>(logits) | (uintptr_t)stride * size) & (4 * size - 1)) == 0;
    const int shift = 62 - bits < 50 ? 62 - bits : 50;
    const SampleArgs a = {logits, stride, logits_type, vocab,  shift, vec4, temperature,
                          top_p,  min_p,  u,           top_k,  tokens,    kept, probs};
    if (vocab <= kSmallVocab) {
        const dim3 grid((unsigned)rows), block(kThreads);
        if (vocab <= kSmallVocab / 2) hipLaunchKernelGGL(sample_small_kernel<8>, grid, block, 0, stream, a);
        else hipLaunchKernelGGL(sample_small_kernel<16>, grid, block, 0, stream, a);
        return hipGetLastError();
    }
    const SampleLayout o = sample_layout(rows, vocab);
    const SampleWs ws = {reinterpret_cast<float *>(workspace + o.tops),
                         reinterpret_cast<float *>(workspace + o.least),
                         reinterpret_cast<u64 *>(workspace + o.mass),
                         reinterpret_cast<u64 *>(workspace + o.chunk_mass),
                         reinterpret_cast<u64 *>(workspace + o.list),
                         reinterpret_cast<Plan *>(workspace + o.plan),
                         reinterpret_cast<uint32_t *>(workspace + o.count),
                         reinterpret_cast<uint32_t *>(workspace + o.chunk_kept),
                         reinterpret_cast<uint32_t *>(workspace + o.listed),
                         o.chunks,
                         o.parts};
    const dim3 grid((unsigned)o.parts, (unsigned)rows);
    hipLaunchKernelGGL(sample_range_kernel, grid, dim3(kScan), 0, stream, a, ws);
    hipLaunchKernelGGL(sample_bins_kernel, grid, dim3(kScan), 0, stream, a, ws);
    // The plans: few workgroups make their row's each, many read it (a histogram
    // is up to 0.4 MB to sum, a launch 2 us).
    if ((int64_t)o.parts * rows <= 128) {
        hipLaunchKernelGGL(sample_collect_kernel<true>, grid, dim3(kScan), 0, stream, a, ws);
    } else {
        hipLaunchKernelGGL(sample_plan_kernel, dim3((unsigned)rows), dim3(kScan), 0, stream, a, ws);
        hipLaunchKernelGGL(sample_collect_kernel<false>, grid, dim3(kScan), 0, stream, a, ws);
    }
    hipLaunchKernelGGL(sample_draw_kernel, dim3((unsigned)rows), dim3(kThreads), 0, stream, a, ws);
    return hipGetLastError();
}

}  // namespace gollek
