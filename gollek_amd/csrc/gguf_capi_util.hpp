// gguf_capi_util.hpp -- what the sources of the C ABI share: the device of a
// call, and whether its buffers lie on one another.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "gollek_hip.h"

namespace gollek {

// A device current for the calls inside, the caller's again afterwards.
class DeviceGuard {
public:
    explicit DeviceGuard(int device) {
        if (hipGetDevice(&before_) != hipSuccess || before_ == device) before_ = -1;
        else if (hipSetDevice(device) != hipSuccess) before_ = -1;
    }
    ~DeviceGuard() {
        if (before_ >= 0) (void)hipSetDevice(before_);
    }
    DeviceGuard(const DeviceGuard &) = delete;
    DeviceGuard &operator=(const DeviceGuard &) = delete;

private:
    int before_ = -1;
};

// The device that holds device memory p (the current one where there is no
// other, or p is not known).
inline int pointer_device(const void *p) {
    static const int devices = [] {
        int n = 0;
        return hipGetDeviceCount(&n) == hipSuccess ? n : 0;
    }();
    int device = 0;
    if (devices > 1) {
        hipPointerAttribute_t at;
        if (hipPointerGetAttributes(&at, p) == hipSuccess && at.type == hipMemoryTypeDevice) return at.device;
        (void)hipGetLastError();
    }
    (void)hipGetDevice(&device);
    return device;
}

inline int element_size(int32_t type) {
    return type == GOLLEK_HIP_F32 ? 4 : type == GOLLEK_HIP_F16 || type == GOLLEK_HIP_BF16 ? 2 : 0;
}

// Whether writing matrix y (m rows of n elements, y_stride apart) changes an
// element of matrix b other than the one at the same place: the same matrix
// is fine, and so are two column ranges of one wider matrix.
inline bool overlaps(const void *y, int64_t y_stride, const void *b, int64_t b_stride, int64_t m, int64_t n, int64_t size) {
    const uintptr_t ya = reinterpret_cast<uintptr_t>(y), ba = reinterpret_cast<uintptr_t>(b);
    const uintptr_t ye = ya + (uintptr_t)(((m - 1) * y_stride + n) * size);
    const uintptr_t be = ba + (uintptr_t)(((m - 1) * b_stride + n) * size);
    if (ye <= ba || be <= ya) return false;
    if (m == 1) return ya != ba;
    if (y_stride != b_stride) return true;
    if (ya == ba) return false;
    const uintptr_t row = (uintptr_t)(y_stride * size), width = (uintptr_t)(n * size);
    const uintptr_t apart = (ya > ba ? ya - ba : ba - ya) % row;
    return !(apart >= width && row - apart >= width);
}

// Whether matrix y and `bytes` bytes at b share a byte (y's gaps between rows counted as y's).
inline bool within(const void *y, int64_t m, int64_t n, int64_t y_stride, int64_t size, const void *b, int64_t bytes) {
    const uintptr_t ya = reinterpret_cast<uintptr_t>(y), ba = reinterpret_cast<uintptr_t>(b);
    return ba < ya + (uintptr_t)(((m - 1) * y_stride + n) * size) && ya < ba + (uintptr_t)bytes;
}

// Whether two stretches of bytes share one (NULL shares none).
inline bool share(const void *a, int64_t a_bytes, const void *b, int64_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a != nullptr && b != nullptr && y < x + (uintptr_t)a_bytes && x < y + (uintptr_t)b_bytes;
}

// Whether two matrices of m rows share a byte: a_bytes (b_bytes) of every row, rows
// a_pitch (b_pitch) bytes apart.  Gaps of rows of one pitch count as free.
inline bool rows_share(const void *a, int64_t a_pitch, int64_t a_bytes, const void *b, int64_t b_pitch, int64_t b_bytes,
                       int64_t m) {
    if (a == nullptr || b == nullptr || m <= 0) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    const uintptr_t xe = x + (uintptr_t)((m - 1) * a_pitch + a_bytes), ye = y + (uintptr_t)((m - 1) * b_pitch + b_bytes);
    if (xe <= y || ye <= x) return false;
    if (m == 1 || a_pitch != b_pitch) return true;
    const uintptr_t pitch = (uintptr_t)a_pitch, apart = y >= x ? (y - x) % pitch : (pitch - (x - y) % pitch) % pitch;
    return !(apart >= (uintptr_t)a_bytes && apart + (uintptr_t)b_bytes <= pitch);
}

}  // namespace gollek
