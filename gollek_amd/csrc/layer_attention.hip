// layer_attention.hip -- attention of one new token a sequence over a paged cache
// of keys and values, on gfx950.
//
//   s_j = scale * q . k_j [softcap * tanh(s_j / softcap)]
//   out = sum_j exp(s_j) v_j / (sum_j exp(s_j) [+ exp(sink)])
//
// in one pass: m a bound of the s so far, l = sum exp(s_j - m), o = sum exp(s_j - m) v_j,
// the last two scaled by exp(m_old - m) when m grows.
//
// A wave takes 32 keys at a time for up to 16 query heads that share them, straight
// from memory to registers:
//   S^T = K Q^T   (two tiles of 16 keys): lane (c, g) = (lane % 16, lane / 16) gets for
//                 query c the keys 4 g .. 4 g + 3 of each tile;
//   O^T += V^T P^T over those 32 keys: the lane's eight weights are, in this order, the
//                 lane's part of the second operand as they stand, when the product's
//                 inner index 8 g + j means key 4 g + j of the first tile (j < 4) or
//                 4 g + j - 4 of the second.
// So weights never cross lanes, and m, l and the accumulators of a query sit in the lanes
// of its column.  For V^T a lane reads the same 8 keys, 8 (or 4) neighbouring dims each,
// and turns them in registers (one v_perm for two elements): fragment i has dim 8 c + i in
// row c.  No LDS in the loop; the next keys are loaded as soon as the scores have used the
// registers, the next values behind the second product.
//
// Weights enter the second product in pieces of the cache's type: three of bf16, together
// an fp32 number's 24 bits, or two of fp16, 22 bits.  Two pieces of bf16 round four times as
// many results otherwise than 64 bits do (0.18 % of them at 700 tokens, three 0.04 %, torch
// in fp32 0.05 %); one puts an error as large as the output's own rounding beside it
// (2.04e-3 against 1.65e-3).  The third costs nothing where bytes count, 3 % of a short
// call (700 tokens 10.7 and 11.0 us) and 4 % where 16 heads read the same keys (37.7 and
// 39.3), as long as the registers of three waves a SIMD suffice for heads of 128.
//
// Bound by bytes: 64 sequences of up to 8192 tokens of 8 heads of 128 219 us (1.37 GB, 6.2
// TB/s; reads alone outrun a copy's 5.0), one of 131072 of 4 heads 41.6 (268 MB, 6.5
// TB/s) and 5.0 for the join.  Short sequences are bound by a step's latency and what a CU
// takes in, a microsecond for the 64 KB of its four waves, whatever the number of steps
// ahead, waves or dims it is asked for: 700 tokens 10.6.
//
// A sequence's tiles are cut into chunks of equal size for workgroups that share the chip
// evenly whatever the lengths are: every workgroup adds up the batch's tiles, takes the
// chunk length from the sum and finds its own sequence and chunk.  Sequences of more than
// one chunk leave (o, m, l) in the workspace, and a second launch joins them.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "layer_kernels.hpp"

namespace gollek {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTile = 32;           // keys of a step
constexpr int kRows = 16;           // query heads of a workgroup
// Tiles of a chunk at least: a step a wave.  (A short sequence is as fast as it has CUs:
// 700 tokens of 8 heads in chunks of 8 tiles 7.0 us, of 4 6.2, of 2 5.7, to which a join
// adds 4.3 to 4.5.)
// Where every CU has a workgroup, kSome: three steps a wave (16 sequences of up to 2048, 8
// heads of 128, with the join: chunks of 4 23.0 us, 8 20.8, 12 20.4, 16 22.1; heads of 256
// 53, 41, 39, 39).
constexpr int kLeast = 4, kSome = 12;
// Workgroups of the kernel that a CU holds, by the registers of its head size.
constexpr int resident(int head_dim) { return head_dim <= 64 ? 4 : head_dim <= 128 ? 3 : head_dim <= 192 ? 2 : 1; }
// Tables of no more tiles than this are not cut at all, which saves the second launch and
// its wait.  With units (key heads of the batch) for fewer than the 256 CUs, us cut and
// whole: 8 heads of 64, 24 tiles 8.5 and 7.7, 32 8.4 and 9.1; of 128, 20 9.3 and 9.1, 24
// 9.3 and 10.1 (but one launch of the caller's less); of 192, 12 10.6 and 9.5, 16 10.7 and
// 11.3; of 256, 12 11.9 and 11.9.  With more, ragged lengths: 256 heads of 128, 32 23.0 and
// 17.9, 48 27.0 and 24.6, 96 51.2 and 49.2; of 256, 48 58 and 51 (a single long sequence
// among them costs a step of 1 to 2 us for every four tiles, hence no further).
constexpr int whole_few(int head_dim) { return resident(head_dim) == 1 ? 12 : 8 * resident(head_dim); }
// (256 here and below is an MI355X's CUs as a number, not asked of the device: a workspace's
// size must not change between the call that asks for it and the one that uses it.)
constexpr int kWholeMany = 48, kFew = 256;
// Many units of few tiles take a wave each, which saves their join through LDS and the
// waves that have no tile: from where workgroups would need more than a round, up to 6
// tiles, or 10 where a CU holds one.  Measured by workgroups and by waves, us: heads of 128,
// one tile, 512 units 5.1 and 5.4, 1024 8.1 and 5.6, 2000 13.1 and 7.7; six tiles 1024 15.9
// and 15.5, 2000 24.2 and 25.5; heads of 256, one tile, 512 11.4 and 8.6, 2000 43 and 17.7;
// six 768 28 and 24, 2000 72 and 55; twelve 768 41 and 43.
constexpr int alone_tiles(int head_dim) { return resident(head_dim) == 1 ? 10 : 6; }
constexpr int alone_units(int head_dim, int64_t tiles) { return 256 * (resident(head_dim) + (tiles <= 2 ? 1 : 2)); }
// Workgroups that a batch is cut into: one for every CU and sequence, up to kTargetMost.
// The chunks of one sequence are all alike, and one round of them does best (131072 tokens
// of 4 heads of 128, main kernel and join: 44.1 + 4.8 us, in 512 44.5 + 5.3, in 768 45.1 +
// 5.8); several sequences' come out between half of T and T, and the more there are the
// shorter the last round should be (two of 65536: 39.1 in 512, 51.8 in 256; 64 of up to
// 8192: 216 in 1536, 225 in 768).
constexpr int kTargetEach = 256, kTargetMost = 1536;
constexpr int kScanMost = 1024;     // sequences whose tiles every workgroup adds up
constexpr float kSlack = 8.0f;      // how far a score may pass m, in powers of two
constexpr float kLog2e = 1.4426950408889634f;

struct AttendPlan {
    int row_tiles;  // workgroups for the query heads of one key head
    bool whole;     // a chunk a sequence
    int slots;      // chunks of a key head that the batch is cut into
    int few;        // chunks of a key head that give every CU a workgroup
    int items;      // chunks at most, and one for every sequence
    int share;      // waves that share a unit (one key head of a chunk, up to kRows query heads)
    bool q_vec;     // queries on 16-byte borders
    // workspace: a chunk's sums, (bound, weight) for each query head, and a sequence's
    // first chunk and how many it has
    float *part_o;
    float2 *part_ml;
    int2 *joins;
};

// A sequence's keys: [begin, length), in tiles from begin's on.
struct Span {
    int begin, length, first, tiles;
};
__device__ __forceinline__ Span span_of(const AttendArgs &a, int length) {
    const int64_t table = a.max_pages << a.kv.page_shift;
    Span s;
    s.length = (int)min((int64_t)max(length, 0), table);
    s.begin = a.window > 0 && s.length > a.window ? s.length - a.window : 0;
    s.first = s.begin / kTile;
    s.tiles = (int)(((int64_t)s.length + kTile - 1) / kTile) - s.first;
    if (s.length == 0) s.tiles = 0;
    return s;
}

__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
// Of the values of the lanes up to each: their sum.  (row_shr 1, 2, 4, 8 within 16
// lanes, then row_bcast 15 and 31.)
template <class T>
__device__ __forceinline__ T prefix_sum(T v) {
    const auto add = [&](int moved) { v += __builtin_bit_cast(T, moved); };
    add(dpp<0x111, 0xF>(__builtin_bit_cast(int, v)));
    add(dpp<0x112, 0xF>(__builtin_bit_cast(int, v)));
    add(dpp<0x114, 0xF>(__builtin_bit_cast(int, v)));
    add(dpp<0x118, 0xF>(__builtin_bit_cast(int, v)));
    add(dpp<0x142, 0xA>(__builtin_bit_cast(int, v)));
    add(dpp<0x143, 0xC>(__builtin_bit_cast(int, v)));
    return v;
}

// What a workgroup works on: chunk `chunk` of `chunks` of a sequence.
struct Item {
    int sequence, length, chunk, chunks;
};

// The sequence that chunk number `item` of the batch belongs to; false past the last.
// By every wave for itself: the batch's tiles are added up, the chunk length T is just
// above tiles / slots, so that all sequences together have at most sequences + slots
// chunks, and the sequences' chunks are counted up to the item.  (The sum is in fp32:
// 22 additions, 2^-19.5 off at most; T is rounded up by more.)
__device__ __forceinline__ bool find_item(const AttendArgs &a, const AttendPlan &p, int item, int lane, Item &it) {
    const int length0 = lane < a.sequences ? a.lengths[lane] : 0;  // (kept: most batches have no more)
    float total = 0.0f;
    for (int s0 = 0; s0 < a.sequences; s0 += 64) {
        const int s = s0 + lane;
        if (s < a.sequences) total += (float)span_of(a, s0 == 0 ? length0 : a.lengths[s]).tiles;
    }
    total = __int_as_float(lane_of(__float_as_int(prefix_sum(total)), 63));
    // (the first bound keeps the chunks within the workspace)
    const int each = max(max(kLeast, (int)fminf(total / (float)p.slots * 1.00001f, 1.0e9f) + 1),
                         min(kSome, (int)fminf(total / (float)p.few, 1.0e9f)));
    int before = 0;
    for (int s0 = 0; s0 < a.sequences; s0 += 64) {
        const int s = s0 + lane;
        const int length = s0 == 0 ? length0 : s < a.sequences ? a.lengths[s] : 0;
        const int n = s < a.sequences ? max(1, (span_of(a, length).tiles + each - 1) / each) : 0;
        const int upto = prefix_sum(n);
        const unsigned long long here = __ballot(before + upto > item);
        if (here != 0) {
            const int l = __builtin_ctzll(here);
            it.sequence = s0 + l;
            it.length = lane_of(length, l);
            it.chunks = lane_of(n, l);
            it.chunk = item - (before + lane_of(upto, l) - it.chunks);
            return true;
        }
        before += lane_of(upto, 63);
    }
    return false;
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c, std::integral_constant<int, kBF16>) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c, std::integral_constant<int, kF16>) {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}

// Two floats rounded to the type, and what that took off.
template <int TYPE>
__device__ __forceinline__ uint32_t round_pair(float &a, float &b) {
    if constexpr (TYPE == kBF16) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        const b2 r = {(__bf16)a, (__bf16)b};
        a -= (float)r[0], b -= (float)r[1];
        return __builtin_bit_cast(uint32_t, r);
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 r = {(_Float16)a, (_Float16)b};
        a -= (float)r[0], b -= (float)r[1];
        return __builtin_bit_cast(uint32_t, r);
    }
}

// Dims of a head as the second product takes them: 16 lanes of kWide0 neighbours,
// then (past 128) 16 of kWide1.
template <int NK>
struct Dims {
    static constexpr int kWide0 = NK <= 2 ? 4 : 8, kWide1 = NK <= 4 ? 0 : NK <= 6 ? 4 : 8;
    static constexpr int kFragments = kWide0 + kWide1, kWords = kFragments / 2;
    static constexpr int kPitch = 16 * kFragments + 4;  // floats of a row in LDS
};

// N neighbouring floats to elements of the output, at any alignment of the element.
template <int N>
__device__ __forceinline__ void store_run(void *p, int type, int64_t i, const float (&v)[N]) {
    if (type == kF32) {
        __builtin_memcpy(static_cast<float *>(p) + i, v, sizeof(v));
    } else {
        uint32_t w[N / 2];
#pragma unroll
        for (int j = 0; j < N / 2; j++) {
            typedef __bf16 b2 __attribute__((ext_vector_type(2)));
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            w[j] = type == kBF16 ? __builtin_bit_cast(uint32_t, b2{(__bf16)v[2 * j], (__bf16)v[2 * j + 1]})
                                 : __builtin_bit_cast(uint32_t, h2{(_Float16)v[2 * j], (_Float16)v[2 * j + 1]});
        }
        __builtin_memcpy(static_cast<uint16_t *>(p) + i, w, sizeof(w));
    }
}

// Values are used once a call: loads that do not stay in the caches.  Keys are too, but an
// instruction takes 64 bytes of each of 16 rows, half a line, and the next one the other
// half: streaming loads fetch it twice (16 sequences of up to 8192, heads of 80: 49 us with
// both streaming, 37 with values alone, 43 with neither; 64 of heads of 128 219, 219, 242).
template <class T>
__device__ __forceinline__ T stream(const T *p) {
    return __builtin_nontemporal_load(p);
}

// Infinite and NaN values.  A piece of a weight may be 0 or below, so an infinite value comes
// out of the second product as NaN where its dim's result is infinite.  Where a sum is NaN
// and its weights' sum is not, the wave that ends it reads the values once more, and they say
// what it is (64 sequences of up to 8192 with an infinity each 410 us in place of 230, one of
// 131072 190 in place of 54; nothing else takes longer).
//
// Of keys first .. end - 1, by a wave: three bits (+infinity, -infinity, NaN among the values)
// for each of the dims 8 piece .. 8 piece + 7 of a lane; piece is its number within `across`,
// the power of two from head_dim / 8 on, and the other lanes take other keys.
template <int TYPE>
__device__ __forceinline__ uint32_t odd_values(const AttendArgs &a, int sequence, int kv_head, int first, int end, int lane,
                                               int across) {
    constexpr uint32_t kExponent = TYPE == kBF16 ? 0x7F80u : 0x7C00u;
    const int32_t *const table = a.page_table + (int64_t)sequence * a.max_pages;
    const int piece = lane & (across - 1), stripes = 64 / across;
    const bool mine = 8 * piece < a.kv.head_dim;
    uint32_t bits = 0;
    constexpr int kAhead = 8;  // keys of a lane in flight
    for (int64_t key0 = first; key0 < end; key0 += kAhead * stripes) {
        int64_t key[kAhead];
        int page[kAhead];
        u32x4 x[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; n++) {
            key[n] = min(key0 + n * stripes + lane / across, (int64_t)end - 1);  // (the last one again: no harm)
            page[n] = table[key[n] >> a.kv.page_shift];
        }
#pragma unroll
        for (int n = 0; n < kAhead; n++) {
            if (page[n] < 0 || page[n] >= a.kv.pages) page[n] = -1;
            const int64_t row = (((int64_t)max(page[n], 0) * a.kv.kv_heads + kv_head) << a.kv.page_shift) +
                                (key[n] & ((1 << a.kv.page_shift) - 1));
            x[n] = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.kv.v) + row * a.kv.head_dim +
                                                    (mine ? 8 * piece : 0));
        }
#pragma unroll
        for (int n = 0; n < kAhead; n++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t h = x[n][j >> 1] >> (16 * (j & 1)) & 0xFFFFu;
                const uint32_t kind = (h & 0x7FFFu) > kExponent ? 4u : h >> 15 != 0 ? 2u : 1u;
                if (page[n] >= 0 && mine && (h & kExponent) == kExponent) bits |= kind << (3 * j);
            }
    }
    for (int m = across; m < 64; m <<= 1) bits |= (uint32_t)__shfl_xor((int)bits, m);
    return bits;
}
__device__ __forceinline__ int piece_lanes(int dim) { return dim <= 8 ? 1 : 1 << (32 - __builtin_clz((unsigned)(dim / 8 - 1))); }
// Dim d's bits of those, for every lane of the wave (which all call it).
__device__ __forceinline__ uint32_t odd_kind(uint32_t bits, int d) { return (uint32_t)__shfl((int)bits, d >> 3) >> (3 * (d & 7)) & 7u; }
// The sum that those bits of a dim stand for; `sum` where they are none.
__device__ __forceinline__ float odd_sum(uint32_t kind, float sum) {
    return kind == 0 ? sum : kind == 1 ? __builtin_inff() : kind == 2 ? -__builtin_inff() : __builtin_nanf("");
}
// A head's sink in powers of two.  One past fp32 there stands for the largest score: it takes
// all weight, and its own stays a number.
__device__ __forceinline__ float sink_of(const AttendArgs &a, int64_t head) {
    const float sink = a.sinks[head] * kLog2e;
    return sink > 3e38f ? 3e38f : sink;
}
// f times a sum; an infinite one stays so where its weights are too small for fp32.
__device__ __forceinline__ float scaled(float f, float sum) { return fabsf(sum) == __builtin_inff() ? sum : f * sum; }

// The keys or values of one step as they stand in registers.
template <int NK>
struct KeyTile {
    u32x4 word[2][NK];
};
template <int NK>
struct ValueTile {
    uint32_t word[8][Dims<NK>::kWords];
};

// TYPE: of cache and queries.  NK: head_dim / 32, rounded up (EXACT: without a rest).
template <int TYPE, int NK, bool EXACT, int SHARE>
__global__ __launch_bounds__(kThreads, NK <= 2 ? 4 : NK <= 4 ? 3 : NK <= 6 ? 2 : 1) void attend_kernel(AttendArgs a, AttendPlan plan) {
    using D = Dims<NK>;
    constexpr std::integral_constant<int, TYPE> type;
    constexpr int kParts = TYPE == kBF16 ? 3 : 2;  // pieces of a weight, of 8 (bf16) or 11 (fp16) bits
    // Weights are exp(s - m) times 2^kLift.  fp16: 2^7, so that all but the smallest are normal
    // numbers (2^15 with the slack, below fp16's largest).  bf16: 2^-kSlack, so that none passes
    // 1 and a value near fp32's largest stays finite times it.
    constexpr float kLift = TYPE == kF16 ? 7.0f : -kSlack;
    const float ninf = -__builtin_inff();

    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int dim = EXACT ? 32 * NK : a.kv.head_dim;
    const int group = a.q_heads / a.kv.kv_heads;
    // Query heads of one key head that take several units read the same keys: as
    // workgroups eight apart, on one XCD; as waves (SHARE 1) side by side.
    int row_tile, unit;
    if constexpr (SHARE > 1) {
        const int id = (int)blockIdx.x;
        row_tile = id / 8 % plan.row_tiles;
        unit = id / (8 * plan.row_tiles) * 8 + id % 8;
    } else {
        const int id = (int)blockIdx.x * kWaves + wave;
        row_tile = id % plan.row_tiles;
        unit = id / plan.row_tiles;
    }
    const int item = unit / a.kv.kv_heads, kv_head = unit % a.kv.kv_heads;
    Item it = {item, 0, 0, 1};
    if (SHARE > 1 && !plan.whole) {
        if (!find_item(a, plan, item, lane, it)) return;
        if (it.chunk == 0 && kv_head == 0 && row_tile == 0 && threadIdx.x == 0)
            plan.joins[it.sequence] = make_int2(item, it.chunks);
    } else {
        if (item >= a.sequences) return;
        it.length = __builtin_amdgcn_readfirstlane(a.lengths[item]);
    }
    const Span span = span_of(a, it.length);
    const int each = (span.tiles + it.chunks - 1) / it.chunks;
    const int tile0 = span.first + it.chunk * each, tile1 = min(tile0 + each, span.first + span.tiles);
    const int row0 = row_tile * kRows, rows = min(kRows, group - row0);
    const int64_t head0 = (int64_t)kv_head * group + row0;

    // queries: row c, dims 32 i + 8 g .. (rows and dims there are none of: 0)
    u32x4 q[NK];
    {
        const uint16_t *const from =
            static_cast<const uint16_t *>(a.q) + it.sequence * a.q_stride + (head0 + (c < rows ? c : 0)) * dim;
        const auto dims = [&](int i) { return EXACT || 32 * i + 8 * g < dim ? 32 * i + 8 * g : 0; };
        if (plan.q_vec) {
#pragma unroll
            for (int i = 0; i < NK; i++) q[i] = *reinterpret_cast<const u32x4 *>(from + dims(i));
        } else {
#pragma unroll
            for (int i = 0; i < NK; i++)
#pragma unroll
                for (int w = 0; w < 4; w++)
                    q[i][w] = (uint32_t)from[dims(i) + 2 * w] | (uint32_t)from[dims(i) + 2 * w + 1] << 16;
        }
    }

    // where a lane reads in a tile of 16 keys, in bytes: its key's row for K, four
    // rows for V (dims past the head's read its first ones, and are not used)
    const bool k_rest = !EXACT && 32 * (NK - 1) + 8 * g >= dim;
    const uint32_t v_col0 = (uint32_t)(D::kWide0 * c < dim ? D::kWide0 * c : 0) * 2;
    const uint32_t v_col1 = (uint32_t)(128 + D::kWide1 * c < dim ? 128 + D::kWide1 * c : 0) * 2;

    const auto table = reinterpret_cast<const __attribute__((address_space(4))) int32_t *>(
        reinterpret_cast<uintptr_t>(a.page_table + (int64_t)it.sequence * a.max_pages));
    // the pages of a tile's two halves (past the length: some page of the sequence)
    const auto pages_of = [&](int tile, int (&page)[2]) {
        page[0] = table[min(kTile * tile, span.length - 1) >> a.kv.page_shift];
        page[1] = table[min(kTile * tile + 16, span.length - 1) >> a.kv.page_shift];
    };
    // byte offset of 16 keys from `key` on, which lie in `page`; -1 where there is none
    const auto place = [&](int page, int key) -> int64_t {
        const bool there = key < span.length && key + 15 >= span.begin && page >= 0 && page < a.kv.pages;
        const int64_t row = ((int64_t)(there ? page : 0) * a.kv.kv_heads + kv_head) << a.kv.page_shift;
        const int64_t at = (row + (key & ((1 << a.kv.page_shift) - 1))) * dim * 2;
        return there ? at : -1;
    };
    const int64_t nowhere = (((int64_t)kv_head) << a.kv.page_shift) * dim * 2;  // (page 0: memory of the cache)

    KeyTile<NK> k;
    ValueTile<NK> v;
    // The first and last row of a half of a tile that are a sequence's; where there are not
    // all, the others' lanes read one of these (a page's other rows are no part of the call).
    const auto rows_of = [&](int key, bool there, int &lo, int &hi) {
        lo = there ? max(span.begin - key, 0) : 0;
        hi = there ? min(span.length - key, 16) - 1 : 0;
    };
    const auto load_keys = [&](const int64_t (&at)[2], int key) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint8_t *const base = static_cast<const uint8_t *>(a.kv.k) + (at[h] < 0 ? nowhere : at[h]);
            int lo, hi;
            rows_of(key + 16 * h, at[h] >= 0, lo, hi);
            const uint32_t row = (uint32_t)(min(max(c, lo), hi) * dim) * 2, off = row + 16 * g;
#pragma unroll
            for (int i = 0; i < NK; i++)
                k.word[h][i] = *reinterpret_cast<const u32x4 *>(base + (i < NK - 1 || !k_rest ? off + 64 * i : row));
        }
    };
    const auto load_run = [&](uint32_t *w, const uint8_t *from, auto WIDE) {
        if constexpr (decltype(WIDE)::value == 8) {
            const u32x4 x = stream(reinterpret_cast<const u32x4 *>(from));
            w[0] = x[0], w[1] = x[1], w[2] = x[2], w[3] = x[3];
        } else if constexpr (decltype(WIDE)::value == 4) {
            const u32x2 x = stream(reinterpret_cast<const u32x2 *>(from));
            w[0] = x[0], w[1] = x[1];
        }
    };
    const auto load_values = [&](const int64_t (&at)[2], int key) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint8_t *const base = static_cast<const uint8_t *>(a.kv.v) + (at[h] < 0 ? nowhere : at[h]);
            int lo, hi;
            rows_of(key + 16 * h, at[h] >= 0, lo, hi);
            uint32_t row[4];
#pragma unroll
            for (int j = 0; j < 4; j++) row[j] = (uint32_t)((4 * g + j) * dim) * 2;
            if (lo > 0 || hi < 15) {
#pragma unroll
                for (int j = 0; j < 4; j++) row[j] = (uint32_t)(min(max(4 * g + j, lo), hi) * dim) * 2;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                load_run(v.word[4 * h + j], base + row[j] + v_col0, std::integral_constant<int, D::kWide0>{});
                load_run(v.word[4 * h + j] + D::kWide0 / 2, base + row[j] + v_col1, std::integral_constant<int, D::kWide1>{});
            }
        }
    };

    f32x4 o[D::kFragments] = {};
    float m = ninf, base = 0.0f, l = 0.0f;  // l of this lane's keys
    const float scale2 = a.scale * kLog2e, cap2 = a.softcap * kLog2e;
    const float turn = a.softcap > 0.0f ? a.scale / a.softcap : 0.0f;

    // One step; MORE: of another one after it, whose keys are loaded when the scores have
    // used the registers, and whose values behind the second product.  (Two copies: a load
    // under a branch would have the wait for this step's values wait for it too.)
    int tile = tile0 + (SHARE > 1 ? wave : 0), page[2];
    int64_t at[2];
    const auto step = [&](auto MORE) {
        constexpr bool more = decltype(MORE)::value;
        f32x4 s[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            s[h] = f32x4{};
            if constexpr (!EXACT) {
                if (k_rest) k.word[h][NK - 1] = u32x4{};
            }
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < NK; i++) s[h] = mfma(k.word[h][i], q[i], s[h], type);
        const int key0 = kTile * tile;
        const bool half[2] = {at[0] >= 0, at[1] >= 0};
        const bool whole = key0 >= span.begin && span.length - key0 >= kTile && half[0] && half[1];
        if constexpr (more) {
            tile += SHARE;
            at[0] = place(page[0], kTile * tile), at[1] = place(page[1], kTile * tile + 16);
            load_keys(at, kTile * tile);
            pages_of(min(tile + SHARE, tile1 - 1), page);
        }
        float x[8];
        if (a.softcap > 0.0f) {
            // (1 - 2 / (1 + exp(2 z)) would be off by 2^-21.5 of the cap, whatever the score: at
            // a cap of 1e6 by all of it.  This one is off by fp32's steps of the score, for 12.3
            // us in place of 11.6 at 700 tokens, 223.5 in place of 222.3 at 64 of up to 8192.)
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = cap2 * tanhf(turn * s[j >> 2][j & 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = scale2 * s[j >> 2][j & 3];
        }
        if (!whole) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int key = key0 + 16 * (j >> 2) + 4 * g + (j & 3);
                const bool in = half[j >> 2] && key >= span.begin && key < span.length;
                x[j] = in ? x[j] : ninf;
#pragma unroll
                for (int w = 0; w < D::kWords; w++) v.word[j][w] = in ? v.word[j][w] : 0;
            }
        }
        float most = x[0];
#pragma unroll
        for (int j = 1; j < 8; j++) most = fmaxf(most, x[j]);
        if (__any(most > m + kSlack)) {
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(fmaxf(most, __shfl_xor(most, 32)), m);
            const float before = m == ninf ? ninf : base;
            m = most;
            base = m == ninf ? 0.0f : m - kLift;
            const float keep = __builtin_amdgcn_exp2f(before - base);
            l *= keep;
#pragma unroll
            for (int i = 0; i < D::kFragments; i++) o[i] *= keep;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] = __builtin_amdgcn_exp2f(x[j] - base);
            l += x[j];
        }
        u32x4 p[kParts];
#pragma unroll
        for (int n = 0; n < kParts; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) p[n][j] = round_pair<TYPE>(x[2 * j], x[2 * j + 1]);
#pragma unroll
        for (int i = 0; i < D::kFragments; i++) {
            u32x4 t;
#pragma unroll
            for (int j = 0; j < 4; j++)
                t[j] = __builtin_amdgcn_perm(v.word[2 * j + 1][i / 2], v.word[2 * j][i / 2],
                                             i % 2 == 0 ? 0x05040100u : 0x07060302u);
#pragma unroll
            for (int n = 0; n < kParts; n++) o[i] = mfma(t, p[n], o[i], type);
        }
        if constexpr (more) load_values(at, kTile * tile);
    };
    if (tile < tile1) {
        pages_of(tile, page);
        at[0] = place(page[0], kTile * tile), at[1] = place(page[1], kTile * tile + 16);
        load_keys(at, kTile * tile);
        load_values(at, kTile * tile);
        pages_of(min(tile + SHARE, tile1 - 1), page);
#pragma unroll
        for (int i = 0; i < NK; i++)
            if (c >= rows || (!EXACT && 32 * i + 8 * g >= dim)) q[i] = u32x4{};
        while (tile + SHARE < tile1) step(std::true_type{});
        step(std::false_type{});
    }

    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const float bound = m == ninf ? ninf : base;
    if constexpr (SHARE == 1) {  // the whole sequence: straight from the accumulators
        float f = 1.0f, total = l;
        if (a.sinks != nullptr && c < rows) {
            const float sink = sink_of(a, head0 + c), up = fmaxf(sink, bound), at1 = up == ninf ? 0.0f : up;
            f = __builtin_amdgcn_exp2f(bound - at1);
            total = l * f + __builtin_amdgcn_exp2f(sink - at1);
        }
        const int64_t row = it.sequence * a.out_stride + (head0 + c) * dim;
        bool odd = false;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const auto put = [&](auto WIDE, int first, int d) {
                constexpr int wide = decltype(WIDE)::value;
                if (d >= dim || c >= rows) return;
                float y[wide];
#pragma unroll
                for (int i = 0; i < wide; i++) {
                    y[i] = total == 0.0f ? 0.0f : f * o[first + i][r] / total;
                    odd |= y[i] != y[i];
                }
                store_run<wide>(a.out, a.out_type, row + d, y);
            };
            put(std::integral_constant<int, D::kWide0>{}, 0, D::kWide0 * (4 * g + r));
            if constexpr (D::kWide1 > 0)
                put(std::integral_constant<int, D::kWide1>{}, D::kWide0, 16 * D::kWide0 + D::kWide1 * (4 * g + r));
        }
        odd = odd && total == total;
        if (__any(odd)) {
            const uint32_t bits = odd_values<TYPE>(a, it.sequence, kv_head, span.begin, span.length, lane, piece_lanes(dim));
#pragma unroll 1
            for (int e = 0; e < 4 * D::kFragments; e++) {
                const int d = e < 4 * D::kWide0 ? 4 * D::kWide0 * g + e : 16 * D::kWide0 + 4 * D::kWide1 * g + e - 4 * D::kWide0;
                const uint32_t kind = odd_kind(bits, d < dim ? d : 0);
                if (odd && d < dim && kind != 0) store_element(a.out, a.out_type, row + d, odd_sum(kind, 0.0f));
            }
        }
        return;
    } else {
        // the waves' sums, rescaled to their common bound, through LDS
        __shared__ __attribute__((aligned(16))) float lds_o[kWaves][kRows * D::kPitch];
        __shared__ float lds_m[kWaves][kRows], lds_l[kWaves][kRows];
        if (g == 0) lds_m[wave][c] = bound, lds_l[wave][c] = l;
        __syncthreads();
        float top = ninf;
#pragma unroll
        for (int w = 0; w < kWaves; w++) top = fmaxf(top, lds_m[w][c]);
        const float keep = __builtin_amdgcn_exp2f(bound - (top == ninf ? 0.0f : top));
        if (c < rows) {
#pragma unroll
            for (int r = 0; r < 4; r++) {  // dims wide * (4 g + r) + i
                float *const to = lds_o[wave] + c * D::kPitch;
#pragma unroll
                for (int i = 0; i < D::kWide0; i++) to[D::kWide0 * (4 * g + r) + i] = keep * o[i][r];
#pragma unroll
                for (int i = 0; i < D::kWide1; i++) to[16 * D::kWide0 + D::kWide1 * (4 * g + r) + i] = keep * o[D::kWide0 + i][r];
            }
        }
        __syncthreads();
        // the sum of element e (kind: what its values' bits say), left where it goes; whether it
        // is NaN over weights that are numbers
        const auto finish = [&](int e, uint32_t kind) -> bool {
            const int r = e / dim, d = e - r * dim;
            float sum = 0.0f, total = 0.0f, most = ninf;
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                sum += lds_o[w][r * D::kPitch + d];
                most = fmaxf(most, lds_m[w][r]);
            }
            const float at0 = most == ninf ? 0.0f : most;
#pragma unroll
            for (int w = 0; w < kWaves; w++) total += lds_l[w][r] * __builtin_amdgcn_exp2f(lds_m[w][r] - at0);
            sum = odd_sum(kind, sum);
            const bool odd = sum != sum && total == total;
            if (it.chunks > 1) {
                const int64_t row = (int64_t)item * a.q_heads + head0 + r;
                plan.part_o[row * dim + d] = sum;
                if (d == 0) plan.part_ml[row] = make_float2(most, total);
            } else {
                if (a.sinks != nullptr) {
                    const float sink = sink_of(a, head0 + r), up = fmaxf(sink, most), at1 = up == ninf ? 0.0f : up;
                    const float f = __builtin_amdgcn_exp2f(at0 - at1);
                    sum = scaled(f, sum);
                    total = total * f + __builtin_amdgcn_exp2f(sink - at1);
                }
                store_element(a.out, a.out_type, it.sequence * a.out_stride + (head0 + r) * dim + d,
                              total == 0.0f ? 0.0f : sum / total);
            }
            return odd;
        };
        bool odd = false;
        for (int e = (int)threadIdx.x; e < rows * dim; e += kThreads) odd |= finish(e, 0);
        if (__any(odd)) {
            const uint32_t bits =
                odd_values<TYPE>(a, it.sequence, kv_head, max(span.begin, kTile * tile0),
                                 (int)min((int64_t)span.length, (int64_t)kTile * tile1), lane, piece_lanes(dim));
            for (int e0 = 64 * wave; e0 < rows * dim; e0 += kThreads) {
                const uint32_t kind = odd_kind(bits, (e0 + lane) % dim);
                if (e0 + lane < rows * dim && kind != 0) (void)finish(e0 + lane, kind);
            }
        }
    }
}

// The chunks of a sequence's query head joined, by one workgroup: groups of `across`
// threads take a chunk at a time, four dims a thread.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void join_kernel(AttendArgs a, AttendPlan plan) {
    constexpr int kThreads = 64 * WAVES, kEach = 4;  // (chunks: at most slots, at most 256 a wave)
    __shared__ float weight[kEach * kThreads], lds_m[WAVES], lds_l[WAVES];
    __shared__ __attribute__((aligned(16))) float lds[4 * kThreads];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, dim = a.kv.head_dim;
    const float ninf = -__builtin_inff();
    const int sequence = (int)blockIdx.x / a.q_heads, head = (int)blockIdx.x % a.q_heads;
    const int2 join = plan.joins[sequence];
    const int64_t row0 = (int64_t)join.x * a.q_heads + head;
    const int chunks = join.y;
    if (chunks <= 1) return;
    const float sink = a.sinks != nullptr ? sink_of(a, head) : ninf;
    float2 ml[kEach];
    float most = sink;
#pragma unroll
    for (int n = 0; n < kEach; n++) {
        const int i = tid + n * kThreads;
        ml[n] = i < chunks ? plan.part_ml[row0 + (int64_t)i * a.q_heads] : make_float2(ninf, 0.0f);
        most = fmaxf(most, ml[n].x);
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) most = fmaxf(most, __shfl_xor(most, m));
    if (lane == 0) lds_m[wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) most = fmaxf(most, lds_m[w]);
    const float at = most == ninf ? 0.0f : most;
    float l = 0.0f;
#pragma unroll
    for (int n = 0; n < kEach; n++) {
        const int i = tid + n * kThreads;
        const float f = __builtin_amdgcn_exp2f(ml[n].x - at);
        if (i < chunks) weight[i] = f;
        l += f * ml[n].y;
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) l += __shfl_xor(l, m);
    if (lane == 0) lds_l[wave] = l;
    __syncthreads();
    const int across = 1 << (32 - __builtin_clz((unsigned)(dim / 4 - 1))), slices = kThreads / across;
    const int slice = tid / across, d0 = 4 * (tid % across);
    f32x4 o = {};
    if (d0 < dim) {
        const float *const from = plan.part_o + row0 * dim + d0;
        const int64_t pitch = (int64_t)a.q_heads * dim;
#pragma unroll 8
        for (int i = slice; i < chunks; i += slices) {
            const f32x4 part = *reinterpret_cast<const f32x4 *>(from + (int64_t)i * pitch);
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] += scaled(weight[i], part[j]);
        }
        *reinterpret_cast<f32x4 *>(lds + slice * dim + d0) = o;
    }
    __syncthreads();
    float total = a.sinks != nullptr ? __builtin_amdgcn_exp2f(sink - at) : 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; w++) total += lds_l[w];
    for (int d = tid; d < dim; d += kThreads) {
        float sum = 0.0f;
        for (int w = 0; w < min(slices, chunks); w++) sum += lds[w * dim + d];
        store_element(a.out, a.out_type, sequence * a.out_stride + (int64_t)head * dim + d, total == 0.0f ? 0.0f : sum / total);
    }
}

AttendPlan make_plan(const KvPages &kv, int sequences, int q_heads, int64_t max_pages, int window) {
    AttendPlan p = {};
    p.row_tiles = (q_heads / kv.kv_heads + kRows - 1) / kRows;
    int64_t tiles = ((max_pages << kv.page_shift) + kTile - 1) / kTile;
    if (window > 0 && tiles > window / kTile + 2) tiles = window / kTile + 2;
    const int64_t per = (int64_t)kv.kv_heads * p.row_tiles, units = sequences * per;
    p.share = tiles <= alone_tiles(kv.head_dim) && units >= alone_units(kv.head_dim, tiles) ? 1 : kWaves;
    // the largest cut, also where this call is not cut: the workspace is asked for by it,
    // and must not shrink where more sequences fall under another rule
    const int n = sequences < kScanMost ? sequences : kScanMost;
    const int target = n < kTargetMost / kTargetEach ? n * kTargetEach : kTargetMost;
    p.slots = (int)(per < target ? target / per : 1);
    p.few = (int)(per < kTargetEach ? kTargetEach / per : 1);
    const int64_t most = n * ((tiles + kLeast - 1) / kLeast);
    // (one slot: no sequence would be cut, its heads are enough)
    p.items = tiles <= whole_few(kv.head_dim) || p.slots == 1 ? 0 : (int)(most < n + p.slots ? most : n + p.slots);
    p.whole = sequences > kScanMost || p.slots == 1 || tiles <= (units < kFew ? whole_few(kv.head_dim) : kWholeMany);
    return p;
}

template <int TYPE>
void launch(int dim, const AttendArgs &a, const AttendPlan &p, unsigned grid, hipStream_t stream) {
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), 0, stream, a, p); };
#define GOLLEK_ATTEND(NK)                                                      \
    case NK:                                                                   \
        if (p.share == 1) {                                                    \
            if (dim == 32 * NK) go(attend_kernel<TYPE, NK, true, 1>);          \
            else go(attend_kernel<TYPE, NK, false, 1>);                        \
        } else {                                                               \
            if (dim == 32 * NK) go(attend_kernel<TYPE, NK, true, kWaves>);    \
            else go(attend_kernel<TYPE, NK, false, kWaves>);                   \
        }                                                                      \
        break
    switch ((dim + 31) / 32) {
        GOLLEK_ATTEND(1);
        GOLLEK_ATTEND(2);
        GOLLEK_ATTEND(3);
        GOLLEK_ATTEND(4);
        GOLLEK_ATTEND(5);
        GOLLEK_ATTEND(6);
        GOLLEK_ATTEND(7);
        GOLLEK_ATTEND(8);
    }
#undef GOLLEK_ATTEND
}

// Bytes of the workspace's parts; p's pointers where there is one.
size_t lay_out(AttendPlan &p, const KvPages &kv, int sequences, int q_heads, uint8_t *workspace) {
    if (p.items == 0) return 0;
    const size_t rows = (size_t)p.items * (size_t)q_heads, o = rows * (size_t)kv.head_dim * sizeof(float);
    const size_t joins = (size_t)(sequences < kScanMost ? sequences : kScanMost) * sizeof(int2);
    p.part_o = reinterpret_cast<float *>(workspace);
    p.part_ml = reinterpret_cast<float2 *>(workspace + o);
    p.joins = reinterpret_cast<int2 *>(workspace + o + rows * sizeof(float2));
    return (o + rows * sizeof(float2) + joins + 255) / 256 * 256;
}

}  // namespace

size_t attend_workspace_bytes(const KvPages &kv, int sequences, int q_heads, int64_t max_pages) {
    AttendPlan p = make_plan(kv, sequences, q_heads, max_pages, 0);
    return lay_out(p, kv, sequences, q_heads, nullptr);
}

hipError_t launch_attend(const AttendArgs &a, uint8_t *workspace, hipStream_t stream) {
    AttendPlan p = make_plan(a.kv, a.sequences, a.q_heads, a.max_pages, a.window);
    (void)lay_out(p, a.kv, a.sequences, a.q_heads, workspace);
    p.q_vec = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * 2)) & 15u) == 0;
    const int64_t units = (int64_t)(p.whole ? a.sequences : p.items) * a.kv.kv_heads;
    // (below 2^24 workgroups, a grid's 2^32 threads: there are fewer rows than that, an uncut
    // unit has one at least, 17 where there are row tiles, and a cut batch has at most 1024 + 1536
    // items of 768 heads)
    const int64_t grid = p.share == 1        ? (units * p.row_tiles + kWaves - 1) / kWaves
                         : p.row_tiles == 1 ? units
                                            : (units + 7) / 8 * 8 * p.row_tiles;
    const int dim = a.kv.head_dim;
    if (a.kv.type == kF16) launch<kF16>(dim, a, p, (unsigned)grid, stream);
    else launch<kBF16>(dim, a, p, (unsigned)grid, stream);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && !p.whole) {
        const dim3 rows((unsigned)(a.sequences * a.q_heads));
        // Waves of a row's join by the chunks it has on the average (most rows of a batch
        // have one, and leave at once), and as many as it may have: 64 sequences of 64 heads
        // by one wave each 4.9 us, four 8.0, sixteen 26.8; one of 64 chunks by one 5.4, four
        // 4.8, sixteen 4.9, two of 128 by four 5.7, sixteen 5.0.
        const auto go = [&](auto kernel, unsigned threads) {
            hipLaunchKernelGGL(kernel, rows, dim3(threads), 0, stream, a, p);
        };
        if (p.slots > 16 * a.sequences || p.slots > 1024) go(join_kernel<16>, 1024);
        else if (p.slots <= 4 * a.sequences && p.slots <= 256) go(join_kernel<1>, 64);
        else go(join_kernel<4>, 256);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace gollek
