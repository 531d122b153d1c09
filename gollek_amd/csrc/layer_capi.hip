// layer_capi.hip -- the C ABI between a decoder layer's products (include/
// gollek_hip.h): norms, rotary positions, the paged key-value cache and its
// attention.  Everything a kernel assumes about its arguments is checked here or
// bounded by the kernel itself (places in the cache, which only the device knows).
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <new>

#include "gguf_capi_util.hpp"
#include "gguf_kernels.hpp"
#include "gollek_hip.h"
#include "layer_kernels.hpp"

constexpr int64_t kRopeMaxDims = 256, kHeadMaxDim = 256;

struct gollek_hip_rope {
    gollek::RopeTable table = {nullptr, 0, false, 1.0f};
    double *turns = nullptr;
    int device = 0;
};

struct gollek_hip_kv_cache {
    gollek::KvPages pages = {};
    int64_t bytes = 0;  // of each array
    int device = 0;
};

namespace {

using gollek::DeviceGuard;
using gollek::element_size;
using gollek::pointer_device;
using gollek::rows_share;
using gollek::share;

constexpr int64_t kInt = 0x7FFFFFFF;
constexpr int64_t kMostElements = (int64_t)1 << 56;  // rows * stride: byte offsets stay in 64 bits

int32_t fail(int32_t code, char *err, size_t err_len, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    gollek::record_status(code, buf);
    if (err != nullptr && err_len > 0) {
        size_t n = strlen(buf);
        if (n >= err_len) n = err_len - 1;
        memcpy(err, buf, n);
        err[n] = '\0';
    }
    return code;
}

int32_t ok(char *err, size_t err_len) {
    gollek::record_status(GOLLEK_HIP_OK, "");
    if (err != nullptr && err_len > 0) err[0] = '\0';
    return GOLLEK_HIP_OK;
}

int32_t hip_fail(hipError_t e, const char *what, char *err, size_t err_len) {
    return fail(e == hipErrorOutOfMemory ? GOLLEK_HIP_ERR_NOMEM : GOLLEK_HIP_ERR_DEVICE, err, err_len, "%s failed: %s",
                what, hipGetErrorString(e));
}

bool aligned(const void *p, uintptr_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// A matrix of a call: `n` elements a row; a stride of 0 becomes n.
struct Rows {
    const char *name;
    const void *p;
    int64_t *stride;
    int64_t n;
    int size;
    int64_t pitch() const { return *stride * size; }
    int64_t bytes() const { return n * size; }
};

int32_t check_rows(Rows &r, int64_t rows, char *err, size_t err_len) {
    if (*r.stride == 0) *r.stride = r.n;
    if (r.p == nullptr) return GOLLEK_HIP_OK;
    if (*r.stride < r.n || *r.stride > kMostElements / (rows > 0 ? rows : 1))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The %s's row stride %lld is not at least %lld, or out of range",
                    r.name, (long long)*r.stride, (long long)r.n);
    if (!aligned(r.p, (uintptr_t)r.size))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The %s is not aligned to its %d-byte elements", r.name, r.size);
    return GOLLEK_HIP_OK;
}

// Whether results `a` share memory with `b` other than element for element (same: allowed).
bool clash(const Rows &a, const Rows &b, int64_t rows, bool same) {
    if (a.p == nullptr || b.p == nullptr) return false;
    if (same && a.p == b.p && a.size == b.size && a.n == b.n && (rows == 1 || *a.stride == *b.stride)) return false;
    return rows_share(a.p, a.pitch(), a.bytes(), b.p, b.pitch(), b.bytes(), rows);
}
bool clash(const Rows &a, int64_t rows, const void *b, int64_t b_bytes) {
    return share(a.p, (rows - 1) * a.pitch() + a.bytes(), b, b_bytes);
}

int32_t overlap(const char *a, const char *b, char *err, size_t err_len) {
    return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The %s overlaps the %s", a, b);
}

}  // namespace

extern "C" {

// ---- norms ------------------------------------------------------------------

static int32_t check_norm(const void *x, int32_t x_type, int64_t rows, int64_t cols, int64_t *x_stride,
                          const float *post_weight, const float *gate, float scale, const void *residual,
                          int64_t *residual_stride, void *hidden, int32_t hidden_type, int64_t *hidden_stride,
                          const float *weight, const float *bias, int32_t kind, float eps, void *y, int32_t y_type,
                          int64_t *y_stride, bool device, char *err, size_t err_len) {
    for (const int32_t t : {x_type, hidden_type, y_type})
        if (element_size(t) == 0)
            return fail(GOLLEK_HIP_ERR_UNSUPPORTED, err, err_len, "Unsupported norm type id: %d (F32, F16 or BF16)", t);
    if (rows < 0 || rows > kInt || cols < 1 || cols > 65536)
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "Rows of %lld x %lld are out of range (at most %lld x 65536)",
                    (long long)rows, (long long)cols, (long long)kInt);
    if (kind != GOLLEK_HIP_NORM_RMS && kind != GOLLEK_HIP_NORM_LAYER)
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "Unknown norm %d", kind);
    if (!isfinite(scale) || !(eps >= 0.0f) || !isfinite(eps))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The norm's scale %g or eps %g is out of range", (double)scale,
                    (double)eps);
    Rows in[] = {{"input", x, x_stride, cols, element_size(x_type)},
                 {"residual", residual, residual_stride, cols, element_size(hidden_type)}};
    Rows out[] = {{"hidden", hidden, hidden_stride, cols, element_size(hidden_type)},
                  {"output", y, y_stride, cols, element_size(y_type)}};
    for (Rows *const set : {in, out})
        for (int i = 0; i < 2; i++) {
            const int32_t rc = check_rows(set[i], rows, err, err_len);
            if (rc != GOLLEK_HIP_OK) return rc;
        }
    const struct {
        const char *name;
        const float *p;
    } vectors[] = {{"post weight", post_weight}, {"gate", gate}, {"weight", weight}, {"bias", bias}};
    for (const auto &v : vectors)
        if (!aligned(v.p, 4)) return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The %s is not aligned to its floats", v.name);
    if (rows == 0) return GOLLEK_HIP_OK;
    if (x == nullptr) return fail(GOLLEK_HIP_ERR_NULL, err, err_len, "input");
    if (hidden == nullptr && y == nullptr) return fail(GOLLEK_HIP_ERR_NULL, err, err_len, "hidden and output");
    if (!device) return GOLLEK_HIP_OK;
    for (const Rows &o : out) {
        for (const Rows &i : in)
            if (clash(o, i, rows, true)) return overlap(o.name, i.name, err, err_len);
        for (const auto &v : vectors)
            if (clash(o, rows, v.p, cols * 4)) return overlap(o.name, v.name, err, err_len);
    }
    if (clash(out[0], out[1], rows, false)) return overlap("hidden", "output", err, err_len);
    return GOLLEK_HIP_OK;
}

int32_t gollek_hip_norm_device(const void *x, int32_t x_type, int64_t rows, int64_t cols, int64_t x_stride,
                               const float *post_weight, const float *gate, float scale, const void *residual,
                               int64_t residual_stride, void *hidden, int32_t hidden_type, int64_t hidden_stride,
                               const float *weight, const float *bias, int32_t kind, float eps, void *y,
                               int32_t y_type, int64_t y_stride, void *stream, char *err, size_t err_len) {
    const int32_t rc =
        check_norm(x, x_type, rows, cols, &x_stride, post_weight, gate, scale, residual, &residual_stride, hidden,
                   hidden_type, &hidden_stride, weight, bias, kind, eps, y, y_type, &y_stride, true, err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    if (rows == 0) return ok(err, err_len);
    const DeviceGuard device(pointer_device(x));
    const hipError_t e = gollek::launch_norm({x, residual, hidden, y, post_weight, gate, weight, bias, x_stride,
                                              residual_stride, hidden_stride, y_stride, rows, (int)cols, x_type,
                                              hidden_type, y_type, kind == GOLLEK_HIP_NORM_LAYER, scale, eps},
                                             static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "norm launch", err, err_len);
    return ok(err, err_len);
}

int32_t gollek_hip_norm(const void *x, int32_t x_type, int64_t rows, int64_t cols, const float *post_weight,
                        const float *gate, float scale, const void *residual, void *hidden, int32_t hidden_type,
                        const float *weight, const float *bias, int32_t kind, float eps, void *y, int32_t y_type,
                        char *err, size_t err_len) {
    int64_t strides[4] = {cols, cols, cols, cols};
    int32_t rc = check_norm(x, x_type, rows, cols, &strides[0], post_weight, gate, scale, residual, &strides[1], hidden,
                            hidden_type, &strides[2], weight, bias, kind, eps, y, y_type, &strides[3], false, err,
                            err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    if (rows == 0) return ok(err, err_len);
    rc = gollek::ready_current_device(err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    // one allocation: x | residual | hidden | y | the four vectors
    const struct {
        const void *in;
        void *out;
        int64_t bytes;
    } each[8] = {{x, nullptr, rows * cols * element_size(x_type)},
                 {residual, nullptr, rows * cols * element_size(hidden_type)},
                 {nullptr, hidden, rows * cols * element_size(hidden_type)},
                 {nullptr, y, rows * cols * element_size(y_type)},
                 {post_weight, nullptr, cols * 4},
                 {gate, nullptr, cols * 4},
                 {weight, nullptr, cols * 4},
                 {bias, nullptr, cols * 4}};
    int64_t total = 0, at[8];
    for (int i = 0; i < 8; i++) {
        at[i] = total;
        if (each[i].in != nullptr || each[i].out != nullptr) total += (each[i].bytes + 255) / 256 * 256;
    }
    uint8_t *d = nullptr, *p[8];
    hipError_t e = hipMalloc(reinterpret_cast<void **>(&d), (size_t)total);
    if (e != hipSuccess) return hip_fail(e, "hipMalloc(norm)", err, err_len);
    for (int i = 0; i < 8; i++) {
        p[i] = each[i].in != nullptr || each[i].out != nullptr ? d + at[i] : nullptr;
        if (e == hipSuccess && each[i].in != nullptr)
            e = hipMemcpy(p[i], each[i].in, (size_t)each[i].bytes, hipMemcpyHostToDevice);
    }
    if (e == hipSuccess)
        e = gollek::launch_norm({p[0], p[1], p[2], p[3], reinterpret_cast<float *>(p[4]), reinterpret_cast<float *>(p[5]),
                                 reinterpret_cast<float *>(p[6]), reinterpret_cast<float *>(p[7]), cols, cols, cols,
                                 cols, rows, (int)cols, x_type, hidden_type, y_type, kind == GOLLEK_HIP_NORM_LAYER,
                                 scale, eps},
                                nullptr);
    for (int i = 2; i < 4; i++)
        if (e == hipSuccess && each[i].out != nullptr)
            e = hipMemcpy(each[i].out, p[i], (size_t)each[i].bytes, hipMemcpyDeviceToHost);
    (void)hipFree(d);
    if (e != hipSuccess) return hip_fail(e, "norm", err, err_len);
    return ok(err, err_len);
}

// ---- rotary positions -------------------------------------------------------

// Radians a position of every pair, in 64 bits.
static int32_t rope_table(int64_t dims, float base, int32_t scaling, float factor, float original_context, float low,
                          float high, float magnitude, const float *factors, double *angles, double *result, char *err,
                          size_t err_len) {
    if (dims < 2 || dims > kRopeMaxDims || dims % 2 != 0)
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "%lld rotary dimensions (an even number from 2 to %lld)",
                    (long long)dims, (long long)kRopeMaxDims);
    if (!(base > 1.0f) || !isfinite(base))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The rotary base %g is not above 1", (double)base);
    if (!(magnitude >= 0.0f) || !isfinite(magnitude))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The rotary magnitude %g is out of range", (double)magnitude);
    if (scaling < GOLLEK_HIP_ROPE_NONE || scaling > GOLLEK_HIP_ROPE_LLAMA3)
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "Unknown rotary scaling %d", scaling);
    if (scaling != GOLLEK_HIP_ROPE_NONE && (!(factor > 0.0f) || !isfinite(factor)))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The rotary scaling factor %g is out of range", (double)factor);
    const bool borders = scaling == GOLLEK_HIP_ROPE_YARN || scaling == GOLLEK_HIP_ROPE_LLAMA3;
    if (borders && (!(original_context > 0.0f) || !isfinite(original_context) || !(low > 0.0f) || !(high > low) ||
                    !isfinite(high)))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The rotary scaling's context %g or borders %g, %g are out of range",
                    (double)original_context, (double)low, (double)high);
    const double two_pi = 2.0 * M_PI;
    double first = 0.0, last = 0.0;
    if (scaling == GOLLEK_HIP_ROPE_YARN) {  // the pairs that turn `high` and `low` times in the context
        const double per = (double)dims / (2.0 * log((double)base));
        first = floor(per * log(original_context / (high * two_pi)));
        last = ceil(per * log(original_context / (low * two_pi)));
        first = first > 0.0 ? first : 0.0;
        last = last < (double)(dims - 1) ? last : (double)(dims - 1);
    }
    for (int64_t i = 0; i < dims / 2; i++) {
        double f = pow((double)base, -2.0 * (double)i / (double)dims);
        if (factors != nullptr) {
            if (!(factors[i] > 0.0f) || !isfinite(factors[i]))
                return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The rotary frequency factor %lld is %g", (long long)i,
                            (double)factors[i]);
            f /= (double)factors[i];
        }
        double keep = 1.0;  // the share of f that is not divided
        if (scaling == GOLLEK_HIP_ROPE_LINEAR) keep = 0.0;
        if (scaling == GOLLEK_HIP_ROPE_YARN) keep = 1.0 - ((double)i - first) / fmax(last - first, 0.001);
        if (scaling == GOLLEK_HIP_ROPE_LLAMA3)
            keep = ((double)original_context * f / two_pi - (double)low) / ((double)high - (double)low);
        keep = fmin(fmax(keep, 0.0), 1.0);
        if (scaling != GOLLEK_HIP_ROPE_NONE) f = f * keep + f / (double)factor * (1.0 - keep);
        if (!isfinite(f)) return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The rotary frequency %lld is not finite", (long long)i);
        angles[i] = f;
    }
    *result = magnitude > 0.0f ? (double)magnitude
              : scaling == GOLLEK_HIP_ROPE_YARN && factor > 1.0f ? 0.1 * log((double)factor) + 1.0
                                                                  : 1.0;
    return GOLLEK_HIP_OK;
}

int32_t gollek_hip_rope_frequencies(int64_t dims, float base, int32_t scaling, float factor, float original_context,
                                    float low, float high, float magnitude, const float *factors, float *frequencies,
                                    float *resulting_magnitude, char *err, size_t err_len) {
    double angles[kRopeMaxDims / 2], result = 1.0;
    const int32_t rc = rope_table(dims, base, scaling, factor, original_context, low, high, magnitude, factors, angles,
                                  &result, err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    if (frequencies != nullptr)
        for (int64_t i = 0; i < dims / 2; i++) frequencies[i] = (float)angles[i];
    if (resulting_magnitude != nullptr) *resulting_magnitude = (float)result;
    return ok(err, err_len);
}

gollek_hip_rope *gollek_hip_rope_create(int32_t layout, int64_t dims, float base, int32_t scaling, float factor,
                                        float original_context, float low, float high, float magnitude,
                                        const float *factors, char *err, size_t err_len) {
    if (layout != GOLLEK_HIP_ROPE_HALF && layout != GOLLEK_HIP_ROPE_INTERLEAVED) {
        fail(GOLLEK_HIP_ERR_ARG, err, err_len, "Unknown rotary layout %d", layout);
        return nullptr;
    }
    double angles[kRopeMaxDims / 2], result = 1.0;
    if (rope_table(dims, base, scaling, factor, original_context, low, high, magnitude, factors, angles, &result, err,
                   err_len) != GOLLEK_HIP_OK)
        return nullptr;
    for (int64_t i = 0; i < dims / 2; i++) angles[i] /= 2.0 * M_PI;
    gollek_hip_rope *const r = new (std::nothrow) gollek_hip_rope;
    if (r == nullptr) {
        fail(GOLLEK_HIP_ERR_NOMEM, err, err_len, "rotary table");
        return nullptr;
    }
    hipError_t e = hipGetDevice(&r->device);
    if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&r->turns), (size_t)(dims / 2) * sizeof(double));
    if (e == hipSuccess) e = hipMemcpy(r->turns, angles, (size_t)(dims / 2) * sizeof(double), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        if (r->turns != nullptr) (void)hipFree(r->turns);
        delete r;
        hip_fail(e, "rotary table", err, err_len);
        return nullptr;
    }
    r->table = {r->turns, (int)dims, layout == GOLLEK_HIP_ROPE_INTERLEAVED, (float)result};
    ok(err, err_len);
    return r;
}

void gollek_hip_rope_free(gollek_hip_rope *r) {
    if (r == nullptr) return;
    {
        const DeviceGuard device(r->device);
        // (the table of a handle that the garbage collector closes while some stream is
        // captured: an ordinary hipFree would break that capture)
        hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
        const bool relaxed = hipThreadExchangeStreamCaptureMode(&mode) == hipSuccess;
        (void)hipFree(r->turns);  // (waits for the device)
        if (relaxed) (void)hipThreadExchangeStreamCaptureMode(&mode);
    }
    delete r;
}

static int32_t check_rope(const gollek_hip_rope *rope, const void *x, int32_t type, int64_t tokens, int64_t heads,
                          int64_t head_dim, int64_t *x_stride, const int32_t *positions, const void *out,
                          int64_t *out_stride, bool device, char *err, size_t err_len) {
    if (rope == nullptr) return fail(GOLLEK_HIP_ERR_NULL, err, err_len, "rotary table");
    if (element_size(type) == 0)
        return fail(GOLLEK_HIP_ERR_UNSUPPORTED, err, err_len, "Unsupported rotary type id: %d (F32, F16 or BF16)", type);
    if (tokens < 0 || tokens > kInt || heads < 1 || heads > 65535 || head_dim < rope->table.dims ||
        head_dim > kHeadMaxDim || head_dim % 2 != 0)
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len,
                    "%lld tokens of %lld heads of %lld are out of range (even heads of %d to %lld)", (long long)tokens,
                    (long long)heads, (long long)head_dim, rope->table.dims, (long long)kHeadMaxDim);
    Rows in = {"input", x, x_stride, heads * head_dim, element_size(type)};
    Rows result = {"output", out, out_stride, heads * head_dim, element_size(type)};
    int32_t rc = check_rows(in, tokens, err, err_len);
    if (rc == GOLLEK_HIP_OK) rc = check_rows(result, tokens, err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    if (!aligned(positions, 4)) return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The positions are not aligned");
    if (tokens == 0) return GOLLEK_HIP_OK;
    if (x == nullptr || out == nullptr || positions == nullptr)
        return fail(GOLLEK_HIP_ERR_NULL, err, err_len, "rotary buffers");
    if (!device) return GOLLEK_HIP_OK;
    if (clash(result, in, tokens, true)) return overlap("output", "input", err, err_len);
    if (clash(result, tokens, positions, tokens * 4)) return overlap("output", "positions", err, err_len);
    if (clash(result, tokens, rope->turns, rope->table.dims * 4)) return overlap("output", "rotary table", err, err_len);
    if (pointer_device(x) != rope->device)
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The rotary table is on another device");
    return GOLLEK_HIP_OK;
}

static gollek::HeadsArgs rope_args(const gollek_hip_rope *rope, const void *x, int32_t type, int64_t tokens,
                                   int64_t heads, int64_t head_dim, int64_t x_stride, const int32_t *positions, void *out,
                                   int64_t out_stride) {
    gollek::HeadsArgs a = {};
    a.q = x;
    a.q_out = out;
    a.q_stride = x_stride;
    a.q_out_stride = out_stride;
    a.rope = rope->table;
    a.positions = positions;
    a.tokens = tokens;
    a.q_heads = (int)heads;
    a.head_dim = (int)head_dim;
    a.type = a.out_type = type;
    return a;
}

int32_t gollek_hip_rope_apply_device(const gollek_hip_rope *rope, const void *x, int32_t type, int64_t tokens,
                                     int64_t heads, int64_t head_dim, int64_t x_stride, const int32_t *positions,
                                     void *out, int64_t out_stride, void *stream, char *err, size_t err_len) {
    const int32_t rc = check_rope(rope, x, type, tokens, heads, head_dim, &x_stride, positions, out, &out_stride, true,
                                  err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    if (tokens == 0) return ok(err, err_len);
    const DeviceGuard device(rope->device);
    const hipError_t e = gollek::launch_heads(
        rope_args(rope, x, type, tokens, heads, head_dim, x_stride, positions, out, out_stride),
        static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "rotary launch", err, err_len);
    return ok(err, err_len);
}

int32_t gollek_hip_rope_apply(const gollek_hip_rope *rope, const void *x, int32_t type, int64_t tokens, int64_t heads,
                              int64_t head_dim, const int32_t *positions, void *out, char *err, size_t err_len) {
    int64_t stride = 0, out_stride = 0;
    const int32_t rc = check_rope(rope, x, type, tokens, heads, head_dim, &stride, positions, out, &out_stride, false,
                                  err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    if (tokens == 0) return ok(err, err_len);
    const DeviceGuard device(rope->device);
    const size_t xn = (size_t)(tokens * heads * head_dim) * element_size(type), pn = (size_t)tokens * 4;
    const size_t xb = (xn + 255) / 256 * 256;
    uint8_t *d = nullptr;
    hipError_t e = hipMalloc(reinterpret_cast<void **>(&d), xb + pn);
    if (e != hipSuccess) return hip_fail(e, "hipMalloc(rotary)", err, err_len);
    e = hipMemcpy(d, x, xn, hipMemcpyHostToDevice);
    if (e == hipSuccess) e = hipMemcpy(d + xb, positions, pn, hipMemcpyHostToDevice);
    if (e == hipSuccess)
        e = gollek::launch_heads(rope_args(rope, d, type, tokens, heads, head_dim, stride,
                                           reinterpret_cast<int32_t *>(d + xb), d, out_stride),
                                 nullptr);
    if (e == hipSuccess) e = hipMemcpy(out, d, xn, hipMemcpyDeviceToHost);
    (void)hipFree(d);
    if (e != hipSuccess) return hip_fail(e, "rotary", err, err_len);
    return ok(err, err_len);
}

// ---- the paged cache --------------------------------------------------------

gollek_hip_kv_cache *gollek_hip_kv_cache_wrap_device(int32_t type, void *k, void *v, int64_t pages, int64_t page_size,
                                                     int64_t kv_heads, int64_t head_dim, char *err, size_t err_len) {
    if (type != GOLLEK_HIP_F16 && type != GOLLEK_HIP_BF16) {
        fail(GOLLEK_HIP_ERR_UNSUPPORTED, err, err_len, "Unsupported cache type id: %d (F16 or BF16)", type);
        return nullptr;
    }
    if (pages < 1 || pages > kInt || page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)) != 0 ||
        kv_heads < 1 || kv_heads > 65535 || head_dim < 8 || head_dim > kHeadMaxDim || head_dim % 8 != 0) {
        fail(GOLLEK_HIP_ERR_ARG, err, err_len,
             "A cache of %lld pages of %lld places, %lld heads of %lld is out of range (pages of 16 to 65536 places, a "
             "power of two; heads of 8 to %lld, a multiple of 8)",
             (long long)pages, (long long)page_size, (long long)kv_heads, (long long)head_dim, (long long)kHeadMaxDim);
        return nullptr;
    }
    // 2^31 pages of 2^40 elements at most: the count could pass 64 bits
    const int64_t page = page_size * kv_heads * head_dim;
    if (page > kMostElements / pages) {
        fail(GOLLEK_HIP_ERR_ARG, err, err_len, "A cache of %lld pages of %lld elements is out of range", (long long)pages,
             (long long)page);
        return nullptr;
    }
    if (k == nullptr || v == nullptr) {
        fail(GOLLEK_HIP_ERR_NULL, err, err_len, "cache arrays");
        return nullptr;
    }
    const int64_t bytes = pages * page * 2;
    if (!aligned(k, 16) || !aligned(v, 16) || share(k, bytes, v, bytes)) {
        fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The cache's keys and values are not 16-byte aligned, or overlap");
        return nullptr;
    }
    gollek_hip_kv_cache *const c = new (std::nothrow) gollek_hip_kv_cache;
    if (c == nullptr) {
        fail(GOLLEK_HIP_ERR_NOMEM, err, err_len, "cache handle");
        return nullptr;
    }
    c->pages = {k, v, pages, __builtin_ctzll((unsigned long long)page_size), (int)kv_heads, (int)head_dim, type};
    c->bytes = bytes;
    c->device = pointer_device(k);
    ok(err, err_len);
    return c;
}

void gollek_hip_kv_cache_free(gollek_hip_kv_cache *c) { delete c; }

static int32_t check_table(const gollek_hip_kv_cache *c, int64_t sequences, int64_t max_pages, char *err, size_t err_len) {
    if (sequences < 0 || sequences > kInt || max_pages < 1 || max_pages > (kInt >> c->pages.page_shift))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "A page table of %lld x %lld pages of %lld places is out of range",
                    (long long)sequences, (long long)max_pages, 1LL << c->pages.page_shift);
    return GOLLEK_HIP_OK;
}

int32_t gollek_hip_kv_append_device(const gollek_hip_kv_cache *cache, const gollek_hip_rope *rope, const void *k,
                                    int64_t k_stride, const void *v, int64_t v_stride, const void *q, int64_t q_heads,
                                    int64_t q_stride, int32_t type, int64_t tokens, const float *q_norm,
                                    const float *k_norm, float eps, const int32_t *positions, const int32_t *sequence,
                                    const int32_t *page_table, int64_t sequences, int64_t max_pages, void *q_out,
                                    int64_t q_out_stride, void *stream, char *err, size_t err_len) {
    if (cache == nullptr) return fail(GOLLEK_HIP_ERR_NULL, err, err_len, "cache");
    if (element_size(type) == 0)
        return fail(GOLLEK_HIP_ERR_UNSUPPORTED, err, err_len, "Unsupported append type id: %d (F32, F16 or BF16)", type);
    const int64_t dim = cache->pages.head_dim, kv = cache->pages.kv_heads;
    if (tokens < 0 || tokens > kInt || q_heads < 0 || q_heads > 65535)
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "%lld tokens of %lld heads are out of range", (long long)tokens,
                    (long long)q_heads);
    int32_t rc = check_table(cache, sequences, max_pages, err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    if (!(eps >= 0.0f) || !isfinite(eps))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The norms' eps %g is out of range", (double)eps);
    if (rope != nullptr && (rope->table.dims > dim || rope->device != cache->device))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len,
                    "The rotary table (%d dimensions) does not fit heads of %lld, or is on another device",
                    rope->table.dims, (long long)dim);
    if (q_heads == 0) q = nullptr;
    const int size = element_size(type);
    Rows in[] = {{"keys", k, &k_stride, kv * dim, size},
                 {"values", v, &v_stride, kv * dim, size},
                 {"queries", q, &q_stride, q_heads * dim, size}};
    Rows out = {"query output", q != nullptr ? q_out : nullptr, &q_out_stride, q_heads * dim, 2};
    for (Rows &r : in) {
        rc = check_rows(r, tokens, err, err_len);
        if (rc != GOLLEK_HIP_OK) return rc;
    }
    rc = check_rows(out, tokens, err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    const struct {
        const char *name;
        const void *p;
        int64_t bytes;
    } small[] = {{"query norm", q_norm, dim * 4},
                 {"key norm", k_norm, dim * 4},
                 {"positions", positions, tokens * 4},
                 {"sequence numbers", sequence, tokens * 4},
                 {"page table", page_table, sequences * max_pages * 4},
                 {"rotary table", rope != nullptr ? rope->turns : nullptr, rope != nullptr ? rope->table.dims * 4 : 0}};
    for (const auto &s : small)
        if (!aligned(s.p, 4)) return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The %s is not aligned", s.name);
    if (tokens == 0) return ok(err, err_len);
    if (k == nullptr || v == nullptr || positions == nullptr || (page_table == nullptr && sequences > 0) ||
        (q_heads > 0 && (q == nullptr || q_out == nullptr)))
        return fail(GOLLEK_HIP_ERR_NULL, err, err_len, "append buffers");
    for (const Rows &r : in) {
        if (clash(r, tokens, cache->pages.k, cache->bytes) || clash(r, tokens, cache->pages.v, cache->bytes))
            return overlap(r.name, "cache", err, err_len);
        if (clash(out, r, tokens, &r == &in[2])) return overlap(out.name, r.name, err, err_len);  // (q_out may be q)
    }
    if (clash(out, tokens, cache->pages.k, cache->bytes) || clash(out, tokens, cache->pages.v, cache->bytes))
        return overlap(out.name, "cache", err, err_len);
    for (const auto &s : small) {
        if (clash(out, tokens, s.p, s.bytes)) return overlap(out.name, s.name, err, err_len);
        if (share(s.p, s.bytes, cache->pages.k, cache->bytes) || share(s.p, s.bytes, cache->pages.v, cache->bytes))
            return overlap(s.name, "cache", err, err_len);
    }
    gollek::HeadsArgs a = {};
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.q_out_stride = q_out_stride;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    if (rope != nullptr) a.rope = rope->table;
    a.kv = cache->pages;
    a.positions = positions;
    a.sequence = sequence;
    a.page_table = page_table;
    a.sequences = sequences;
    a.max_pages = max_pages;
    a.tokens = tokens;
    a.q_heads = (int)q_heads;
    a.head_dim = (int)dim;
    a.type = type;
    a.out_type = cache->pages.type;
    const DeviceGuard device(cache->device);
    const hipError_t e = gollek::launch_heads(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "append launch", err, err_len);
    return ok(err, err_len);
}

static int32_t check_attention(const gollek_hip_kv_cache *cache, int64_t sequences, int64_t q_heads, int64_t max_pages,
                               char *err, size_t err_len) {
    const int32_t rc = check_table(cache, sequences, max_pages, err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    if (sequences > 65535 || q_heads < 1 || q_heads > 65535 || q_heads % cache->pages.kv_heads != 0 ||
        sequences * q_heads >= (int64_t)1 << 24)
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len,
                    "%lld sequences of %lld heads over %d heads of the cache are out of range", (long long)sequences,
                    (long long)q_heads, cache->pages.kv_heads);
    return GOLLEK_HIP_OK;
}

int64_t gollek_hip_attention_workspace_bytes(const gollek_hip_kv_cache *cache, int64_t sequences, int64_t q_heads,
                                             int64_t max_pages) {
    if (cache == nullptr || check_attention(cache, sequences, q_heads, max_pages, nullptr, 0) != GOLLEK_HIP_OK) return -1;
    if (sequences == 0) return 0;
    return (int64_t)gollek::attend_workspace_bytes(cache->pages, (int)sequences, (int)q_heads, max_pages);
}

int32_t gollek_hip_attention_device(const gollek_hip_kv_cache *cache, const void *q, int64_t q_stride,
                                    int64_t sequences, int64_t q_heads, const int32_t *lengths,
                                    const int32_t *page_table, int64_t max_pages, float scale, float softcap,
                                    int64_t window, const float *sinks, void *out, int32_t out_type,
                                    int64_t out_stride, void *workspace, int64_t workspace_bytes, void *stream,
                                    char *err, size_t err_len) {
    if (cache == nullptr) return fail(GOLLEK_HIP_ERR_NULL, err, err_len, "cache");
    if (element_size(out_type) == 0)
        return fail(GOLLEK_HIP_ERR_UNSUPPORTED, err, err_len, "Unsupported attention type id: %d (F32, F16 or BF16)",
                    out_type);
    int32_t rc = check_attention(cache, sequences, q_heads, max_pages, err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    // (the kernel takes scale / softcap and both times log2 e: none may overflow)
    if (!(fabsf(scale) <= 1e15f) || !(softcap == 0.0f || (softcap >= 1e-15f && softcap <= 1e15f)) || window < 0)
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The attention's scale %g, cap %g or window %lld is out of range",
                    (double)scale, (double)softcap, (long long)window);
    const int64_t dim = cache->pages.head_dim;
    Rows in = {"queries", q, &q_stride, q_heads * dim, 2};
    Rows result = {"output", out, &out_stride, q_heads * dim, element_size(out_type)};
    rc = check_rows(in, sequences, err, err_len);
    if (rc == GOLLEK_HIP_OK) rc = check_rows(result, sequences, err, err_len);
    if (rc != GOLLEK_HIP_OK) return rc;
    if (!aligned(lengths, 4) || !aligned(page_table, 4) || !aligned(sinks, 4))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "The lengths, page table or sinks are not aligned");
    if (sequences == 0) return ok(err, err_len);
    if (q == nullptr || lengths == nullptr || page_table == nullptr || out == nullptr)
        return fail(GOLLEK_HIP_ERR_NULL, err, err_len, "attention buffers");
    const int64_t need = gollek_hip_attention_workspace_bytes(cache, sequences, q_heads, max_pages);
    if (need > 0 && workspace == nullptr) return fail(GOLLEK_HIP_ERR_NULL, err, err_len, "attention workspace");
    if (workspace_bytes < need || !aligned(workspace, 256))
        return fail(GOLLEK_HIP_ERR_ARG, err, err_len, "Workspace of %lld bytes (256-byte aligned) needed, got %lld",
                    (long long)need, (long long)workspace_bytes);
    const struct {
        const char *name;
        const void *p;
        int64_t bytes;
    } read[] = {{"queries", q, (sequences - 1) * in.pitch() + in.bytes()},
                {"keys", cache->pages.k, cache->bytes},
                {"values", cache->pages.v, cache->bytes},
                {"lengths", lengths, sequences * 4},
                {"page table", page_table, sequences * max_pages * 4},
                {"sinks", sinks, q_heads * 4}};
    if (clash(result, in, sequences, false)) return overlap("output", "queries", err, err_len);
    for (const auto &r : read) {
        if (&r != &read[0] && clash(result, sequences, r.p, r.bytes)) return overlap("output", r.name, err, err_len);
        if (share(r.p, r.bytes, workspace, need)) return overlap("workspace", r.name, err, err_len);
    }
    if (clash(result, sequences, workspace, need)) return overlap("output", "workspace", err, err_len);
    const DeviceGuard device(cache->device);
    const hipError_t e = gollek::launch_attend(
        {cache->pages, q, out, q_stride, out_stride, lengths, page_table, sinks, max_pages, (int)sequences, (int)q_heads,
         out_type, (int)(window > kInt ? kInt : window), scale, softcap},
        static_cast<uint8_t *>(workspace), static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, "attention launch", err, err_len);
    return ok(err, err_len);
}

}  // extern "C"
