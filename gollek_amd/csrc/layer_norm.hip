// layer_norm.hip -- the norms around a block, on gfx950.
//
//   b = post ? N(x) * post : x;  h = residual + scale * gate * b  -> hidden
//   y = N(h) * weight + bias;  N(v) = v / sqrt(mean(v^2) + eps), or of v - mean(v)
//
// One workgroup a row at a time; the row stays in registers in fp32 from the first
// load to the last store, so x and the residual are read once and nothing is read
// back.  A thread has PER pieces of eight neighbouring elements, loaded as 16 bytes at
// whatever alignment the row has (odd lengths and strides included).
//
// Bound by bytes: 8192 x 4096 bf16 with a norm behind the block, gate and residual 54 to
// 61 us for 268 MB (4.4 to 5.0 TB/s; a copy 5.0).  There the four vectors would be as many
// bytes again from L2 if every row loaded them: a workgroup keeps them in registers and
// walks over rows, the next row's loads in flight while it reduces this one.  Few rows are
// bound by a launch and one chain of loads and sums: 1 x 4096 3.2 us (one piece a thread,
// so that all loads of the row go out at once; 13.0 with 16 elements one by one).
#include <hip/hip_runtime.h>

#include "gguf_kernels.hpp"  // device_cus
#include "layer_kernels.hpp"

namespace gollek {
namespace {

constexpr int kPiece = 8;

template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xF, false));
}
// The wave's sum, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
    v = dpp_add<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8, then row_bcast 15, 31: lane 63 has it
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    v = dpp_add<0x143, 0xC>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Sums over the workgroup.  Every one has the next of three LDS rows, so one barrier
// does: a row is written again only two barriers after it was read.
struct BlockSum {
    float (*lds)[16];
    int next = 0;
    __device__ __forceinline__ float operator()(float v) {
        v = wave_sum(v);
        const int waves = (int)blockDim.x >> 6;
        if (waves == 1) return v;
        float *const row = lds[next];
        next = next == 2 ? 0 : next + 1;
        if ((threadIdx.x & 63) == 0) row[threadIdx.x >> 6] = v;
        __syncthreads();
        float sum = row[0];
        for (int w = 1; w < waves; w++) sum += row[w];
        return sum;
    }
};

// Eight elements of SIZE bytes as they stand in memory, at any alignment of the element;
// `type` tells fp16 from bf16.  (By size, not by type: eight kernels in place of 27.)
template <int SIZE>
struct Piece {
    uint32_t bits[kPiece * SIZE / 4];
    __device__ __forceinline__ void load(const void *p, int64_t i) {
        __builtin_memcpy(bits, static_cast<const uint8_t *>(p) + i * SIZE, sizeof(bits));
    }
    __device__ __forceinline__ void get(float (&v)[kPiece], int type) const {
        if constexpr (SIZE == 4) {
#pragma unroll
            for (int j = 0; j < kPiece; j++) v[j] = __uint_as_float(bits[j]);
        } else if (type == kBF16) {
#pragma unroll
            for (int j = 0; j < kPiece; j++)
                v[j] = __uint_as_float((j & 1) ? bits[j >> 1] & 0xFFFF0000u : bits[j >> 1] << 16);
        } else {
#pragma unroll
            for (int j = 0; j < kPiece; j++)
                v[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(bits[j >> 1] >> (16 * (j & 1))));
        }
    }
    __device__ __forceinline__ void set(const float (&v)[kPiece], int type) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        if constexpr (SIZE == 4) {
#pragma unroll
            for (int j = 0; j < kPiece; j++) bits[j] = __float_as_uint(v[j]);
        } else if (type == kBF16) {
#pragma unroll
            for (int j = 0; j < 4; j++) bits[j] = __builtin_bit_cast(uint32_t, b2{(__bf16)v[2 * j], (__bf16)v[2 * j + 1]});
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                bits[j] = __builtin_bit_cast(uint32_t, h2{(_Float16)v[2 * j], (_Float16)v[2 * j + 1]});
        }
    }
    __device__ __forceinline__ void store(void *p, int64_t i) const {
        __builtin_memcpy(static_cast<uint8_t *>(p) + i * SIZE, bits, sizeof(bits));
    }
};

// Elements i .. i + 7 of a row that starts at `row`, 0 past `cols`.
template <int SIZE>
__device__ __forceinline__ void fetch(Piece<SIZE> &p, const void *from, int type, int64_t row, int i, int cols) {
    if (i + kPiece <= cols) {
        p.load(from, row + i);
    } else {
        float v[kPiece];
        for (int j = 0; j < kPiece; j++) v[j] = i + j < cols ? load_element(from, type, row + i + j) : 0.0f;
        p.set(v, type);
    }
}
template <int SIZE>
__device__ __forceinline__ void leave(const float (&v)[kPiece], void *to, int type, int64_t row, int i, int cols) {
    if (i + kPiece <= cols) {
        Piece<SIZE> p;
        p.set(v, type);
        p.store(to, row + i);
    } else {
        for (int j = 0; j < kPiece; j++)
            if (i + j < cols) store_element(to, type, row + i + j, v[j]);
    }
}

// X, H, Y: element sizes of x, of hidden and the residual, and of y.  HOLD: the vectors
// stay in registers from row to row, and the next row is loaded before this one is
// computed; without, every piece is loaded where it is used (rows of many pieces).
template <int X, int H, int Y, int PER, int THREADS, bool HOLD>
__global__ __launch_bounds__(THREADS) void norm_kernel(NormArgs a) {
    __shared__ float lds[3][16];
    BlockSum block_sum = {lds};
    const int cols = a.cols;
    const float over = 1.0f / (float)cols;
    const auto at = [&](int c) { return kPiece * (c * (int)blockDim.x + (int)threadIdx.x); };
    constexpr int kVectors = HOLD ? PER : 1;
    Piece<4> post[kVectors], gate[kVectors], weight[kVectors], bias[kVectors];
    Piece<X> x[kVectors];
    Piece<H> residual[kVectors];
    int64_t row = blockIdx.x;
    const auto load_x = [&](int64_t row, int c) {
        if (at(c) < cols) fetch(x[c % kVectors], a.x, a.x_type, row * a.x_stride, at(c), cols);
    };
    const auto load_residual = [&](int64_t row, int c) {
        if (a.residual != nullptr && at(c) < cols)
            fetch(residual[c % kVectors], a.residual, a.hidden_type, row * a.residual_stride, at(c), cols);
    };
    const auto load_vector = [&](Piece<4>(&v)[kVectors], const float *p, int c) {
        if (p != nullptr && at(c) < cols) fetch(v[c % kVectors], p, kF32, 0, at(c), cols);
    };
    if constexpr (HOLD) {
#pragma unroll
        for (int c = 0; c < PER; c++) load_x(row, c);
#pragma unroll
        for (int c = 0; c < PER; c++) {
            load_residual(row, c);
            load_vector(post, a.post, c);
            load_vector(gate, a.gate, c);
            load_vector(weight, a.weight, c);
            load_vector(bias, a.bias, c);
        }
    }
    float h[PER][kPiece];
    // h <- N(h), elements past the row 0 again
    const auto normalise = [&] {
        float sum = 0.0f;
        if (a.layer) {
#pragma unroll
            for (int c = 0; c < PER; c++)
#pragma unroll
                for (int j = 0; j < kPiece; j++) sum += h[c][j];
            const float mean = block_sum(sum) * over;
#pragma unroll
            for (int c = 0; c < PER; c++)
#pragma unroll
                for (int j = 0; j < kPiece; j++) h[c][j] = at(c) + j < cols ? h[c][j] - mean : 0.0f;
            sum = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < PER; c++)
#pragma unroll
            for (int j = 0; j < kPiece; j++) sum += h[c][j] * h[c][j];
        const float r = 1.0f / sqrtf(block_sum(sum) * over + a.eps);
#pragma unroll
        for (int c = 0; c < PER; c++)
#pragma unroll
            for (int j = 0; j < kPiece; j++) h[c][j] *= r;
    };
    const auto times = [&](float (&v)[kPiece], const Piece<4> &by) {
#pragma unroll
        for (int j = 0; j < kPiece; j++) v[j] *= __uint_as_float(by.bits[j]);
    };
    while (true) {
        const int64_t next = row + gridDim.x;
#pragma unroll
        for (int c = 0; c < PER; c++) {
            if (at(c) < cols) {
                if constexpr (!HOLD) load_x(row, c);
                x[c % kVectors].get(h[c], a.x_type);
            } else {
#pragma unroll
                for (int j = 0; j < kPiece; j++) h[c][j] = 0.0f;
            }
        }
        if constexpr (HOLD) {
            if (next < a.rows) {
#pragma unroll
                for (int c = 0; c < PER; c++) load_x(next, c);
            }
        }
        if (a.post != nullptr) {
            normalise();
#pragma unroll
            for (int c = 0; c < PER; c++) {
                if (at(c) >= cols) continue;
                if constexpr (!HOLD) load_vector(post, a.post, c);
                times(h[c], post[c % kVectors]);
            }
        }
#pragma unroll
        for (int c = 0; c < PER; c++) {
            if (at(c) >= cols) continue;
            if constexpr (!HOLD) load_vector(gate, a.gate, c), load_residual(row, c);
#pragma unroll
            for (int j = 0; j < kPiece; j++) h[c][j] *= a.scale;
            if (a.gate != nullptr) times(h[c], gate[c % kVectors]);
            if (a.residual != nullptr) {
                float add[kPiece];
                residual[c % kVectors].get(add, a.hidden_type);
#pragma unroll
                for (int j = 0; j < kPiece; j++) h[c][j] += add[j];
            }
            if (a.hidden != nullptr) leave<H>(h[c], a.hidden, a.hidden_type, row * a.hidden_stride, at(c), cols);
        }
        if constexpr (HOLD) {
            if (next < a.rows) {
#pragma unroll
                for (int c = 0; c < PER; c++) load_residual(next, c);
            }
        }
        if (a.y != nullptr) {
            normalise();
#pragma unroll
            for (int c = 0; c < PER; c++) {
                if (at(c) >= cols) continue;
                if constexpr (!HOLD) load_vector(weight, a.weight, c), load_vector(bias, a.bias, c);
                if (a.weight != nullptr) times(h[c], weight[c % kVectors]);
                if (a.bias != nullptr) {
#pragma unroll
                    for (int j = 0; j < kPiece; j++) h[c][j] += __uint_as_float(bias[c % kVectors].bits[j]);
                }
                leave<Y>(h[c], a.y, a.y_type, row * a.y_stride, at(c), cols);
            }
        }
        if (next >= a.rows) break;
        row = next;
    }
}

template <int X, int H, int Y>
void launch(const NormArgs &a, hipStream_t stream) {
    // Up to one row a CU: as many threads as the row has pieces.  More: two pieces a thread
    // and rows in turn, 1024 threads a CU (8192 x 4096: 58 us; one piece 61 to 79, 768
    // threads a CU 68, a workgroup a row 72).  Longer rows, past what registers hold beside
    // the vectors: nothing held (1000 x 14336 31 us).
    const int pieces = (a.cols + kPiece - 1) / kPiece, cus = device_cus();
    const auto go = [&](auto kernel, int per, int resident) {
        const int threads = ((pieces + per - 1) / per + 63) / 64 * 64;
        const int64_t most = (int64_t)cus * (resident / threads);
        hipLaunchKernelGGL(kernel, dim3((unsigned)(a.rows < most ? a.rows : most)), dim3((unsigned)threads), 0, stream, a);
    };
    if (pieces <= 1024 && a.rows <= cus) go(norm_kernel<X, H, Y, 1, 1024, true>, 1, 2048);
    else if (pieces <= 1024) go(norm_kernel<X, H, Y, 2, 512, true>, 2, 1024);
    else if (pieces <= 2048) go(norm_kernel<X, H, Y, 2, 1024, false>, 2, 2048);
    else go(norm_kernel<X, H, Y, 8, 1024, false>, 8, 2048);
}
template <int X, int H>
void launch(const NormArgs &a, hipStream_t stream) {
    if (a.y_type == kF32) launch<X, H, 4>(a, stream);
    else launch<X, H, 2>(a, stream);
}
template <int X>
void launch(const NormArgs &a, hipStream_t stream) {
    if (a.hidden_type == kF32) launch<X, 4>(a, stream);
    else launch<X, 2>(a, stream);
}

}  // namespace

hipError_t launch_norm(const NormArgs &a, hipStream_t stream) {
    if (a.x_type == kF32) launch<4>(a, stream);
    else launch<2>(a, stream);
    return hipGetLastError();
}

}  // namespace gollek
