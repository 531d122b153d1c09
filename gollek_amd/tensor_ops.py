"""Host-side mirror of gollek's GgufTensorOps facade over libgollek_hip.so.

The reference facade is RT/GgufTensorOps.java (RT/ = runner/gguf/
gollek-gguf-core/src/main/java/tech/kayys/gollek/gguf/runtime/): static
dequantizeRow / dotRow / matVec / matVecParallel / matVecRows over a
(GGUFModel, GGUFTensorInfo) pair whose bytes live in an mmapped file.  Here a
GgufTensor carries the same (name, shape, type id, bytes) facts and uploads its
bytes once to a device handle, the way the Java drop-in would key a handle by
(model, tensor).  Calls have the reference's names, argument meaning and
exceptions:

    NullPointerError       <- GOLLEK_HIP_ERR_NULL      (Objects.requireNonNull)
    IllegalArgumentError   <- GOLLEK_HIP_ERR_ARG       (IllegalArgumentException)
    UnsupportedOperationError <- GOLLEK_HIP_ERR_UNSUPPORTED
    DeviceError            <- GOLLEK_HIP_ERR_DEVICE / NOMEM

Every call goes through the C ABI; there is no host fallback.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field

import numpy as np

from . import _native

BLOCK = {_native.Q4_0: (32, 18), _native.Q8_0: (32, 34), _native.Q4_K: (256, 144),
         _native.Q5_K: (256, 176), _native.Q6_K: (256, 210)}
TYPE_NAMES = {_native.Q4_0: "Q4_0", _native.Q8_0: "Q8_0", _native.Q4_K: "Q4_K",
              _native.Q5_K: "Q5_K", _native.Q6_K: "Q6_K"}


class GgufHipError(RuntimeError):
    code = 0


class NullPointerError(GgufHipError, TypeError):
    code = _native.ERR_NULL


class IllegalArgumentError(GgufHipError, ValueError):
    code = _native.ERR_ARG


class UnsupportedOperationError(GgufHipError, NotImplementedError):
    code = _native.ERR_UNSUPPORTED


class DeviceError(GgufHipError):
    code = _native.ERR_DEVICE


_BY_CODE = {
    _native.ERR_NULL: NullPointerError,
    _native.ERR_ARG: IllegalArgumentError,
    _native.ERR_UNSUPPORTED: UnsupportedOperationError,
    _native.ERR_DEVICE: DeviceError,
    _native.ERR_NOMEM: DeviceError,
}


def check(rc: int, err: _native.ErrBuf) -> None:
    if rc != _native.OK:
        raise _BY_CODE.get(rc, GgufHipError)(err.text or f"status {rc}")


def row_bytes_for(type_id: int, cols: int) -> int:
    bs, bb = BLOCK[type_id]
    return cols // bs * bb


def init(device: int = 0) -> None:
    lib = _native.load()
    err = _native.ErrBuf()
    check(lib.gollek_hip_init(device, err.buf, err.size), err)


def set_option(key: str, value: int) -> None:
    """Test-only kernel-family switch (gollek_hip_testing_set_option): the
    parity tests force each GEMV / MoE kernel family onto shapes another one
    is picked for.  Not part of the reference's interface."""
    lib = _native.load()
    err = _native.ErrBuf()
    check(lib.gollek_hip_testing_set_option(key.encode(), int(value), err.buf, err.size), err)


@dataclass
class GgufTensor:
    """GGUFTensorInfo(name, shape, typeId, ...) plus its bytes.

    shape[0] is the column count (contiguous); the remaining dimensions form
    the rows (RT/GgufTensorOps.java:621-630)."""

    name: str
    shape: tuple[int, ...]
    type_id: int
    data: np.ndarray  # uint8, rows * row_bytes
    _handle: int | None = field(default=None, repr=False)
    # set for tensors of a GgufFile: the handle comes from the file upload
    _file: "GgufFile | None" = field(default=None, repr=False)
    _index: int = field(default=-1, repr=False)

    @property
    def columns(self) -> int:
        return int(self.shape[0])

    @property
    def rows(self) -> int:
        r = 1
        for d in self.shape[1:]:
            r *= int(d)
        return r

    @property
    def row_bytes(self) -> int:
        bs, bb = BLOCK.get(self.type_id, (1, 1))
        return self.columns // bs * bb

    def handle(self) -> int:
        """Device handle, created on first use (the prepared-cache analogue)."""
        if self._handle is None and self._file is not None:
            self._handle = self._file.upload(self._index)
        if self._handle is None:
            lib = _native.load()
            err = _native.ErrBuf()
            buf = np.ascontiguousarray(self.data, dtype=np.uint8)
            h = lib.gollek_hip_weight_upload(self.type_id, buf.ctypes.data, self.rows,
                                             self.columns, self.row_bytes, err.buf, err.size)
            if not h:
                raise _BY_CODE.get(lib.gollek_hip_last_status(), GgufHipError)(err.text)
            self._handle = h
        return self._handle

    def prepare(self) -> None:
        """Build the handle's prepared mat-vec layout (gollek_hip_weight_prepare;
        the reference builds its prepared matrices at model load)."""
        err = _native.ErrBuf()
        check(_native.load().gollek_hip_weight_prepare(self.handle(), err.buf, err.size), err)

    def unprepare(self) -> None:
        """Free the prepared layout (gollek_hip_weight_unprepare); full
        mat-vecs read the GGUF bytes again (the prepared-cache clear)."""
        if self._handle is not None:
            err = _native.ErrBuf()
            check(_native.load().gollek_hip_weight_unprepare(self._handle, err.buf, err.size), err)

    def compact(self) -> None:
        """Keep only the prepared layout (gollek_hip_weight_compact): the
        packed bytes are held once; GEMM and MoE then raise
        UnsupportedOperationError."""
        err = _native.ErrBuf()
        check(_native.load().gollek_hip_weight_compact(self.handle(), err.buf, err.size), err)

    def close(self) -> None:
        if self._handle is not None:
            _native.load().gollek_hip_weight_free(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _f32_out(arr, name: str) -> np.ndarray:
    if arr is None:
        raise NullPointerError(name)
    if not (isinstance(arr, np.ndarray) and arr.dtype == np.float32 and arr.flags.c_contiguous):
        raise IllegalArgumentError(f"{name} must be a contiguous float32 array")
    return arr


def _f32_in(arr, name: str) -> np.ndarray:
    if arr is None:
        raise NullPointerError(name)
    return np.ascontiguousarray(arr, dtype=np.float32)


def dequantize_row(tensor: GgufTensor, row: int, dst: np.ndarray) -> None:
    """GgufTensorOps.dequantizeRow (RT/GgufTensorOps.java:636-642)."""
    if tensor is None:
        raise NullPointerError("tensor")
    dst = _f32_out(dst, "dst")
    lib = _native.load()
    err = _native.ErrBuf()
    if dst.size < tensor.columns:
        raise IllegalArgumentError(
            f"Vector length {dst.size} is smaller than columns {tensor.columns}")
    check(lib.gollek_hip_dequantize_rows(tensor.handle(), int(row), 1, dst.ctypes.data,
                                         tensor.columns, err.buf, err.size), err)


def dequantize_rows(tensor: GgufTensor, row0: int, nrows: int) -> np.ndarray:
    """Bit-exact dequantization of a row range (for parity checks)."""
    out = np.empty((max(nrows, 0), tensor.columns), dtype=np.float32)
    lib = _native.load()
    err = _native.ErrBuf()
    check(lib.gollek_hip_dequantize_rows(tensor.handle(), int(row0), int(nrows),
                                         out.ctypes.data, out.size, err.buf, err.size), err)
    return out


def dot_row(tensor: GgufTensor, row: int, vector) -> float:
    """GgufTensorOps.dotRow (RT/GgufTensorOps.java:644-650)."""
    if tensor is None:
        raise NullPointerError("tensor")
    x = _f32_in(vector, "vector")
    out = np.zeros(1, dtype=np.float32)
    lib = _native.load()
    err = _native.ErrBuf()
    check(lib.gollek_hip_dot_row(tensor.handle(), int(row), x.ctypes.data, x.size,
                                 out.ctypes.data, err.buf, err.size), err)
    return float(out[0])


def mat_vec_rows(tensor: GgufTensor, vector, output: np.ndarray, row_count: int,
                 parallel: bool = True) -> None:
    """GgufTensorOps.matVecRows (RT/GgufTensorOps.java:666-674).

    `parallel` is accepted for signature parity; the GPU always runs all
    rows concurrently."""
    if tensor is None:
        raise NullPointerError("tensor")
    x = _f32_in(vector, "vector")
    y = _f32_out(output, "output")
    lib = _native.load()
    err = _native.ErrBuf()
    check(lib.gollek_hip_matvec_rows(tensor.handle(), x.ctypes.data, x.size, y.ctypes.data,
                                     y.size, int(row_count), err.buf, err.size), err)


def mat_vec(tensor: GgufTensor, vector, output: np.ndarray) -> None:
    """GgufTensorOps.matVec (RT/GgufTensorOps.java:658-660)."""
    if tensor is None:
        raise NullPointerError("tensor")
    mat_vec_rows(tensor, vector, output, tensor.rows, False)


def mat_vec_parallel(tensor: GgufTensor, vector, output: np.ndarray) -> None:
    """GgufTensorOps.matVecParallel (RT/GgufTensorOps.java:662-664)."""
    if tensor is None:
        raise NullPointerError("tensor")
    mat_vec_rows(tensor, vector, output, tensor.rows, True)


# ---- GGUF files -------------------------------------------------------------

@dataclass(frozen=True)
class GgufTensorInfo:
    """GC/loader/GGUFTensorInfo.java:8-14 (GC/ = runner/gguf/gollek-gguf-core/
    src/main/java/tech/kayys/gollek/gguf/): name, shape (shape[0] contiguous),
    ggml type id, offset from the data start, size in bytes."""

    name: str
    shape: tuple[int, ...]
    type_id: int
    offset: int
    size_in_bytes: int


class GgufFile:
    """A GGUF file opened through the native parser: the facts GGUFModel holds
    (GC/loader/GGUFParser.java:17-62: version, tensor infos, data start) and a
    device upload per tensor (GC/runtime/GgufTensorData.java:97-104's range
    check, then the weight upload).  Metadata values other than
    general.alignment are not kept."""

    def __init__(self, path):
        lib = _native.load()
        err = _native.ErrBuf()
        self.path = str(path)
        h = lib.gollek_hip_gguf_open(self.path.encode(), err.buf, err.size)
        if not h:
            raise _BY_CODE.get(lib.gollek_hip_last_status(), GgufHipError)(err.text)
        self._h = h
        v, nt, nkv, al, ds, fb = (ctypes.c_int32(), ctypes.c_int64(), ctypes.c_int64(),
                                  ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64())
        lib.gollek_hip_gguf_info(h, *(ctypes.byref(o) for o in (v, nt, nkv, al, ds, fb)))
        self.version, self.n_kv, self.alignment = v.value, nkv.value, al.value
        self.data_start, self.file_bytes = ds.value, fb.value
        self.tensors: list[GgufTensorInfo] = [self._info(i) for i in range(nt.value)]
        self._map = None

    def _info(self, index: int) -> GgufTensorInfo:
        lib = _native.load()
        name = ctypes.create_string_buffer(4096)
        tid, nd = ctypes.c_int32(), ctypes.c_int32()
        dims = (ctypes.c_int64 * 8)()
        off, size = ctypes.c_int64(), ctypes.c_int64()
        rc = lib.gollek_hip_gguf_tensor(self._h, index, name, 4096, ctypes.byref(tid),
                                        ctypes.byref(nd), dims, ctypes.byref(off),
                                        ctypes.byref(size))
        if rc != 0:
            raise _BY_CODE.get(rc, GgufHipError)(f"tensor index {index}")
        return GgufTensorInfo(name.value.decode("utf-8", "replace"),
                              tuple(int(dims[d]) for d in range(nd.value)), tid.value,
                              off.value, size.value)

    def find(self, name: str) -> int:
        """Index of the tensor called `name`, or -1."""
        return int(_native.load().gollek_hip_gguf_find(self._h, name.encode()))

    def upload(self, index: int) -> int:
        """A new device weight handle holding tensor `index` (caller frees it)."""
        lib = _native.load()
        err = _native.ErrBuf()
        h = lib.gollek_hip_gguf_upload(self._h, index, err.buf, err.size)
        if not h:
            raise _BY_CODE.get(lib.gollek_hip_last_status(), GgufHipError)(err.text)
        return h

    def tensor(self, name: str) -> GgufTensor:
        """GgufTensor for `name` whose bytes are a read-only view of the file
        (empty where they fall outside it) and whose handle comes from
        upload()."""
        index = self.find(name)
        if index < 0:
            raise IllegalArgumentError(f"Tensor not found: {name}")
        info = self.tensors[index]
        if self._map is None:
            self._map = np.memmap(self.path, dtype=np.uint8, mode="r")
        start = self.data_start + info.offset
        data = self._map[start:start + info.size_in_bytes] if start >= 0 else self._map[:0]
        return GgufTensor(info.name, info.shape, info.type_id, data, _file=self, _index=index)

    def close(self) -> None:
        if self._h:
            _native.load().gollek_hip_gguf_close(self._h)
            self._h = None
        self._map = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- device-pointer entry points (inputs already resident in HBM) ---------

# activations of linear()
ACT_NONE = 0
ACT_RELU = 1
ACT_SILU = 2
ACT_GELU = 3
ACT_GELU_TANH = 4

class DeviceWeight:
    """A handle over GGUF bytes already in device memory (borrowed)."""

    def __init__(self, type_id: int, device_ptr: int, rows: int, cols: int):
        lib = _native.load()
        err = _native.ErrBuf()
        self.type_id, self.rows, self.cols = type_id, rows, cols
        self.row_bytes = row_bytes_for(type_id, cols)
        h = lib.gollek_hip_weight_wrap_device(type_id, ctypes.c_void_p(device_ptr), rows, cols,
                                              self.row_bytes, err.buf, err.size)
        if not h:
            raise _BY_CODE.get(lib.gollek_hip_last_status(), GgufHipError)(err.text)
        self.handle = h

    def prepare(self) -> None:
        """Build the handle's prepared mat-vec layout (gollek_hip_weight_prepare)."""
        err = _native.ErrBuf()
        check(_native.load().gollek_hip_weight_prepare(self.handle, err.buf, err.size), err)

    def unprepare(self) -> None:
        """Free the prepared layout (gollek_hip_weight_unprepare)."""
        err = _native.ErrBuf()
        check(_native.load().gollek_hip_weight_unprepare(self.handle, err.buf, err.size), err)

    def compact(self) -> None:
        """Keep only the prepared layout (gollek_hip_weight_compact)."""
        err = _native.ErrBuf()
        check(_native.load().gollek_hip_weight_compact(self.handle, err.buf, err.size), err)

    def close(self) -> None:
        if self.handle:
            _native.load().gollek_hip_weight_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def matvec(self, x_ptr: int, y_ptr: int, row_count: int | None = None,
               stream: int = 0) -> None:
        lib = _native.load()
        err = _native.ErrBuf()
        rc = lib.gollek_hip_matvec_device(self.handle, ctypes.c_void_p(x_ptr),
                                          ctypes.c_void_p(y_ptr),
                                          self.rows if row_count is None else row_count,
                                          ctypes.c_void_p(stream), err.buf, err.size)
        check(rc, err)

    def dequantize(self, row0: int, nrows: int, dst_ptr: int, stream: int = 0) -> None:
        lib = _native.load()
        err = _native.ErrBuf()
        rc = lib.gollek_hip_dequantize_rows_device(self.handle, row0, nrows,
                                                   ctypes.c_void_p(dst_ptr),
                                                   ctypes.c_void_p(stream), err.buf, err.size)
        check(rc, err)

    def gemm_bf16(self, x_ptr: int, m: int, y_ptr: int, stream: int = 0) -> None:
        lib = _native.load()
        err = _native.ErrBuf()
        rc = lib.gollek_hip_gemm_bf16_device(self.handle, ctypes.c_void_p(x_ptr), m,
                                             ctypes.c_void_p(y_ptr), ctypes.c_void_p(stream),
                                             err.buf, err.size)
        check(rc, err)


    def linear_workspace_bytes(self, m: int) -> int:
        """Device workspace with which linear() of m rows splits K as far as it
        pays (0: never)."""
        return int(_native.load().gollek_hip_linear_workspace_bytes(self.handle, m))

    def linear(self, x_ptr: int, m: int, y_ptr: int, y_type: int, *, y_stride: int = 0, bias_ptr: int = 0,
               activation: int = ACT_NONE, mul_ptr: int = 0, mul_stride: int = 0, residual_ptr: int = 0,
               residual_stride: int = 0, ws_ptr: int = 0, ws_bytes: int = 0, stream: int = 0) -> None:
        """Y = act(X W^T + bias) * mul + residual (gollek_hip_linear_device): x
        bf16 (m, cols), y / mul / residual of y_type with row strides (0:
        packed), bias float32.  mul and residual may be y itself."""
        err = _native.err_buf()
        check(_native.load().gollek_hip_linear_device(self.handle, x_ptr, m, bias_ptr, activation, mul_ptr,
                                                      mul_stride, residual_ptr, residual_stride, y_ptr, y_type,
                                                      y_stride, ws_ptr, ws_bytes, stream, err.buf, err.size), err)


_LINEAR_DTYPES = {_native.F32: np.float32, _native.F16: np.float16, _native.BF16: np.uint16}


def linear(tensor: GgufTensor, x_bf16: np.ndarray, y_type: int = _native.F32, *, bias=None,
           activation: int = ACT_NONE, mul=None, residual=None) -> np.ndarray:
    """act(X W^T + bias) * mul + residual on host arrays: x_bf16 (m, columns)
    uint16 bf16 bit patterns, bias (rows,) float32, mul and residual (m, rows) of
    y_type (BF16 as uint16 bit patterns) -> (m, rows) of y_type."""
    if tensor is None:
        raise NullPointerError("tensor")
    if x_bf16 is None:
        raise NullPointerError("input")
    if y_type not in _LINEAR_DTYPES:
        raise UnsupportedOperationError(f"Unsupported linear output type id: {y_type} (F32, F16 or BF16)")
    x = np.ascontiguousarray(x_bf16, dtype=np.uint16)
    if x.ndim != 2 or x.shape[1] != tensor.columns:
        raise IllegalArgumentError(f"input must be (m, {tensor.columns})")
    m, dtype = x.shape[0], _LINEAR_DTYPES[y_type]

    def operand(a, name, shape, dt):
        if a is None:
            return None
        a = np.ascontiguousarray(a)
        if a.shape != shape or a.dtype != dt:
            raise IllegalArgumentError(f"{name} must be {shape} of {np.dtype(dt).name}")
        return a

    b = operand(bias, "bias", (tensor.rows,), np.float32)
    mu = operand(mul, "mul", (m, tensor.rows), dtype)
    re = operand(residual, "residual", (m, tensor.rows), dtype)
    y = np.empty((m, tensor.rows), dtype)
    at = [None if a is None else a.ctypes.data for a in (b, mu, re)]
    err = _native.ErrBuf()
    check(_native.load().gollek_hip_linear(tensor.handle(), x.ctypes.data, x.size, m, at[0], activation, at[1], at[2],
                                           y.ctypes.data, y_type, y.size, err.buf, err.size), err)
    return y


def gemm_bf16(tensor: GgufTensor, x_bf16: np.ndarray, output: np.ndarray) -> None:
    """Y = X W^T for a Q8_0, Q4_0 or Q4_K tensor: x_bf16 (m, columns) uint16 bf16 bit patterns,
    output (m, rows) float32.  The reference runs m matVecRows calls instead
    (RT/GgufTensorOps.java:666-674)."""
    if tensor is None:
        raise NullPointerError("tensor")
    if x_bf16 is None:
        raise NullPointerError("input")
    x = np.ascontiguousarray(x_bf16, dtype=np.uint16)
    y = _f32_out(output, "output")
    m = x.shape[0] if x.ndim == 2 else x.size // max(tensor.columns, 1)
    lib = _native.load()
    err = _native.ErrBuf()
    check(lib.gollek_hip_gemm_bf16(tensor.handle(), x.ctypes.data, x.size, int(m), y.ctypes.data,
                                   y.size, err.buf, err.size), err)


def moe_grouped(gate: GgufTensor, up: GgufTensor, down: GgufTensor, n_experts: int, x, ids,
                weights) -> np.ndarray:
    """Grouped MoE expert FFN over Q4_0 / Q8_0 / Q4_K / Q5_K / Q6_K experts
    (gate, up and down may differ; the expert loop of MoeForwardPass.computeAccel,
    runner/safetensor/gollek-safetensor-engine/src/main/java/tech/kayys/gollek/
    safetensor/engine/generation/moe/MoeForwardPass.java:217-240): x (tokens,
    hidden) float32, ids (tokens, top_k) int32, weights (tokens, top_k) float32
    -> (tokens, hidden) float32."""
    for name, t in (("gate", gate), ("up", up), ("down", down)):
        if t is None:
            raise NullPointerError(name)
    xv = np.ascontiguousarray(x, dtype=np.float32)
    iv = np.ascontiguousarray(ids, dtype=np.int32)
    wv = np.ascontiguousarray(weights, dtype=np.float32)
    tokens, top_k = iv.shape
    out = np.zeros((tokens, gate.columns), dtype=np.float32)
    lib = _native.load()
    err = _native.ErrBuf()
    check(lib.gollek_hip_moe_grouped(gate.handle(), up.handle(), down.handle(), n_experts,
                                     xv.ctypes.data, tokens, iv.ctypes.data, wv.ctypes.data,
                                     top_k, out.ctypes.data, out.size, err.buf, err.size), err)
    return out


def moe_workspace_bytes(tokens: int, top_k: int, hidden: int, inter: int, n_experts: int) -> int:
    return int(_native.load().gollek_hip_moe_workspace_bytes(tokens, top_k, hidden, inter,
                                                             n_experts))


def moe_grouped_device(gate: DeviceWeight, up: DeviceWeight, down: DeviceWeight, n_experts: int,
                       x_ptr: int, ids_ptr: int, w_ptr: int, tokens: int, top_k: int,
                       out_ptr: int, ws_ptr: int, ws_bytes: int, stream: int = 0) -> None:
    lib = _native.load()
    err = _native.ErrBuf()
    V = ctypes.c_void_p
    rc = lib.gollek_hip_moe_grouped_device(gate.handle, up.handle, down.handle, n_experts,
                                           V(x_ptr), V(ids_ptr), V(w_ptr), tokens, top_k,
                                           V(out_ptr), V(ws_ptr), ws_bytes, V(stream), err.buf,
                                           err.size)
    check(rc, err)


# ---- MoE router and routed block ---------------------------------------------

ROUTER_SOFTMAX = 0
ROUTER_SIGMOID = 1


def router_scoring(model_type: str | None) -> int:
    """The reference's choice (MoeForwardPass.java:174-175): sigmoid when the
    model type contains "qwen" or "moe", softmax otherwise."""
    mt = model_type or ""
    return ROUTER_SIGMOID if ("qwen" in mt or "moe" in mt) else ROUTER_SOFTMAX


def moe_select_topk(logits, top_k: int, scoring: int):
    """Router probabilities and renormalised top-k (MoeForwardPass.java:174-203
    with selectTopK :286-306) on the GPU: logits (tokens, n_experts) float32
    -> ids (tokens, top_k) int32, weights (tokens, top_k) float32."""
    lv = np.ascontiguousarray(logits, dtype=np.float32)
    if lv.ndim != 2:
        raise IllegalArgumentError("logits must be (tokens, n_experts)")
    tokens, n_experts = lv.shape
    ids = np.zeros((tokens, top_k), np.int32)
    w = np.zeros((tokens, top_k), np.float32)
    lib = _native.load()
    err = _native.ErrBuf()
    check(lib.gollek_hip_moe_select_topk(lv.ctypes.data, tokens, n_experts, top_k, scoring,
                                         ids.ctypes.data, w.ctypes.data, err.buf, err.size), err)
    return ids, w


def moe_block(gate: GgufTensor, up: GgufTensor, down: GgufTensor, n_experts: int, x, logits,
              top_k: int, scoring: int) -> np.ndarray:
    """The routed MoE block (MoeForwardPass.java:174-240 after the router
    linear): router on `logits`, then the grouped expert FFN (expert types as
    moe_grouped)."""
    for name, t in (("gate", gate), ("up", up), ("down", down)):
        if t is None:
            raise NullPointerError(name)
    xv = np.ascontiguousarray(x, dtype=np.float32)
    lv = np.ascontiguousarray(logits, dtype=np.float32)
    tokens = xv.shape[0]
    out = np.zeros((tokens, gate.columns), dtype=np.float32)
    lib = _native.load()
    err = _native.ErrBuf()
    check(lib.gollek_hip_moe_block(gate.handle(), up.handle(), down.handle(), n_experts,
                                   xv.ctypes.data, tokens, lv.ctypes.data, top_k, scoring,
                                   out.ctypes.data, out.size, err.buf, err.size), err)
    return out


def moe_block_device(gate: DeviceWeight, up: DeviceWeight, down: DeviceWeight, n_experts: int,
                     x_ptr: int, logits_ptr: int, tokens: int, top_k: int, scoring: int,
                     ids_ptr: int, w_ptr: int, out_ptr: int, ws_ptr: int, ws_bytes: int,
                     stream: int = 0) -> None:
    lib = _native.load()
    err = _native.ErrBuf()
    V = ctypes.c_void_p
    rc = lib.gollek_hip_moe_block_device(gate.handle, up.handle, down.handle, n_experts,
                                         V(x_ptr), V(logits_ptr), tokens, top_k, scoring,
                                         V(ids_ptr), V(w_ptr), V(out_ptr), V(ws_ptr), ws_bytes,
                                         V(stream), err.buf, err.size)
    check(rc, err)


def _logits(a):
    """A host array of logits as it is passed on, and its element type: float16
    and bf16 bit patterns (uint16) as they are, every other type as float32."""
    a = np.ascontiguousarray(a)
    if a.dtype == np.float16:
        return a, _native.F16
    if a.dtype == np.uint16:
        return a, _native.BF16
    return np.ascontiguousarray(a, dtype=np.float32), _native.F32


def moe_route(logits, top_k: int, scoring: int, *, bias=None, n_groups: int = 1, top_groups: int = 1,
              group_top: int = 1, renormalize: bool = True, scale: float = 1.0):
    """Routing with a balancing bias and groups (gollek_hip_moe_route) on host
    arrays: logits (tokens, n_experts) float32, float16 or uint16 bf16 bit
    patterns (as linear returns them) -> ids (tokens, top_k) int32, weights
    (tokens, top_k) float32."""
    if logits is None:
        raise NullPointerError("logits")
    lv, kind = _logits(logits)
    if lv.ndim != 2:
        raise IllegalArgumentError("logits must be (tokens, n_experts)")
    tokens, n_experts = lv.shape
    bv = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
    if bv is not None and bv.shape != (n_experts,):
        raise IllegalArgumentError(f"bias must be ({n_experts},)")
    ids = np.zeros((tokens, max(top_k, 0)), np.int32)
    w = np.zeros((tokens, max(top_k, 0)), np.float32)
    err = _native.ErrBuf()
    check(_native.load().gollek_hip_moe_route(lv.ctypes.data, kind, tokens, n_experts,
                                              None if bv is None else bv.ctypes.data, scoring, n_groups, top_groups,
                                              group_top, top_k, int(renormalize), scale, ids.ctypes.data,
                                              w.ctypes.data, err.buf, err.size), err)
    return ids, w


def moe_route_device(logits_ptr: int, logits_type: int, tokens: int, n_experts: int, top_k: int, scoring: int,
                     ids_ptr: int, w_ptr: int, *, bias_ptr: int = 0, n_groups: int = 1, top_groups: int = 1,
                     group_top: int = 1, renormalize: bool = True, scale: float = 1.0, stream: int = 0) -> None:
    err = _native.err_buf()
    check(_native.load().gollek_hip_moe_route_device(logits_ptr, logits_type, tokens, n_experts, bias_ptr, scoring,
                                                     n_groups, top_groups, group_top, top_k, renormalize, scale,
                                                     ids_ptr, w_ptr, stream, err.buf, err.size), err)


def moe_block_routed_device(gate: DeviceWeight, up: DeviceWeight, down: DeviceWeight, n_experts: int, x_ptr: int,
                            logits_ptr: int, logits_type: int, tokens: int, top_k: int, scoring: int, ids_ptr: int,
                            w_ptr: int, out_ptr: int, ws_ptr: int, ws_bytes: int, *, bias_ptr: int = 0,
                            n_groups: int = 1, top_groups: int = 1, group_top: int = 1, renormalize: bool = True,
                            scale: float = 1.0, stream: int = 0) -> None:
    """moe_route_device followed by moe_grouped_device on one stream
    (gollek_hip_moe_block_routed_device)."""
    err = _native.err_buf()
    check(_native.load().gollek_hip_moe_block_routed_device(
        gate.handle, up.handle, down.handle, n_experts, x_ptr, logits_ptr, logits_type, tokens, bias_ptr, scoring,
        n_groups, top_groups, group_top, top_k, renormalize, scale, ids_ptr, w_ptr, out_ptr, ws_ptr, ws_bytes, stream,
        err.buf, err.size), err)


def moe_shared_expert(gate: GgufTensor, up: GgufTensor, down: GgufTensor, x, out,
                      gate_inp=None) -> np.ndarray:
    """The shared expert added to the routed output `out` (MoeForwardPass.java:
    240-247, runSharedExpert :418-426, resolveSharedExpertGate :428-442):
    out[t] + g_t * down(silu(gate x_t) * (up x_t)) with g_t = sigmoid(x_t .
    gate_inp) (1 without gate_inp).  Returns the new output; `out` is not
    modified."""
    for name, t in (("gate", gate), ("up", up), ("down", down)):
        if t is None:
            raise NullPointerError(name)
    xv = np.ascontiguousarray(x, dtype=np.float32)
    res = np.array(out, dtype=np.float32, order="C", copy=True)
    gi = None if gate_inp is None else np.ascontiguousarray(gate_inp, dtype=np.float32)
    lib = _native.load()
    err = _native.ErrBuf()
    V = ctypes.c_void_p
    check(lib.gollek_hip_moe_shared_expert(gate.handle(), up.handle(), down.handle(),
                                           V(None) if gi is None else V(gi.ctypes.data),
                                           V(xv.ctypes.data), xv.shape[0], V(res.ctypes.data),
                                           res.size, err.buf, err.size), err)
    return res


def moe_shared_workspace_bytes(tokens: int, hidden: int, inter: int) -> int:
    return int(_native.load().gollek_hip_moe_shared_workspace_bytes(tokens, hidden, inter))


def moe_shared_expert_device(gate: DeviceWeight, up: DeviceWeight, down: DeviceWeight,
                             gate_inp_ptr: int, x_ptr: int, tokens: int, out_ptr: int, ws_ptr: int,
                             ws_bytes: int, stream: int = 0) -> None:
    lib = _native.load()
    err = _native.ErrBuf()
    V = ctypes.c_void_p
    rc = lib.gollek_hip_moe_shared_expert_device(gate.handle, up.handle, down.handle,
                                                 V(gate_inp_ptr or None), V(x_ptr), tokens,
                                                 V(out_ptr), V(ws_ptr), ws_bytes, V(stream),
                                                 err.buf, err.size)
    check(rc, err)


# ---- sampling ------------------------------------------------------------------

def sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token per row of logits (gollek_hip_sample) on host arrays: logits
    (rows, vocab) float32, float16 or uint16 bf16 bit patterns (as linear returns
    them), u (rows,) the random numbers, settings scalars or (rows,) arrays
    (None: off, temperature 1) -> tokens int32, probs float32, kept int32, each
    (rows,)."""
    if logits is None:
        raise NullPointerError("logits")
    if u is None:
        raise NullPointerError("u")
    lv, kind = _logits(logits)
    if lv.ndim != 2:
        raise IllegalArgumentError("logits must be (rows, vocab)")
    rows, vocab = lv.shape

    def per_row(v, name, dtype):
        if v is None:
            return None
        a = np.asarray(v, dtype=dtype)
        if a.ndim == 0:
            a = np.full(rows, a, dtype)
        if a.shape != (rows,):
            raise IllegalArgumentError(f"{name} must be a number or ({rows},)")
        return np.ascontiguousarray(a)

    args = [per_row(v, n, t) for v, n, t in ((temperature, "temperature", np.float32), (top_k, "top_k", np.int32),
                                             (top_p, "top_p", np.float32), (min_p, "min_p", np.float32),
                                             (u, "u", np.float32))]
    tokens, probs, kept = np.empty(rows, np.int32), np.empty(rows, np.float32), np.empty(rows, np.int32)
    err = _native.ErrBuf()
    check(_native.load().gollek_hip_sample(lv.ctypes.data, kind, rows, vocab,
                                           *(None if a is None else a.ctypes.data for a in args), tokens.ctypes.data,
                                           probs.ctypes.data, kept.ctypes.data, err.buf, err.size), err)
    return tokens, probs, kept


def sample_workspace_bytes(rows: int, vocab: int) -> int:
    return int(_native.load().gollek_hip_sample_workspace_bytes(rows, vocab))


def sample_device(logits_ptr: int, logits_type: int, rows: int, vocab: int, u_ptr: int, tokens_ptr: int, *,
                  logits_stride: int = 0, temperature_ptr: int = 0, top_k_ptr: int = 0, top_p_ptr: int = 0,
                  min_p_ptr: int = 0, probs_ptr: int = 0, kept_ptr: int = 0, ws_ptr: int = 0, ws_bytes: int = 0,
                  stream: int = 0) -> None:
    err = _native.err_buf()
    check(_native.load().gollek_hip_sample_device(logits_ptr, logits_type, rows, vocab, logits_stride,
                                                  temperature_ptr, top_k_ptr, top_p_ptr, min_p_ptr, u_ptr, tokens_ptr,
                                                  probs_ptr, kept_ptr, ws_ptr, ws_bytes, stream, err.buf, err.size),
          err)


def next_token(lm_head: GgufTensor, vector, u: float, *, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
               min_p: float = 0.0):
    """The lm_head's mat-vec of `vector` (floats, or uint16 bf16 bit patterns as
    linear returns them) and a token sampled from it (gollek_hip_next_token; the
    logits stay on the device) -> token, prob, kept."""
    if lm_head is None:
        raise NullPointerError("tensor")
    if getattr(vector, "dtype", None) == np.uint16:
        vector = (np.asarray(vector, np.uint32) << 16).view(np.float32)  # exact
    x = _f32_in(vector, "vector")
    token, prob, kept = ctypes.c_int32(), ctypes.c_float(), ctypes.c_int32()
    err = _native.err_buf()
    check(_native.load().gollek_hip_next_token(lm_head.handle(), x.ctypes.data, x.size, temperature, top_k, top_p,
                                               min_p, u, ctypes.byref(token), ctypes.byref(prob), ctypes.byref(kept),
                                               err.buf, err.size), err)
    return token.value, prob.value, kept.value


# ---- between the products of a decoder layer -----------------------------------

NORM_RMS = 0
NORM_LAYER = 1
ROPE_HALF = 0
ROPE_INTERLEAVED = 1
ROPE_NONE = 0
ROPE_LINEAR = 1
ROPE_YARN = 2
ROPE_LLAMA3 = 3


def _typed(a, name):
    """A host array as it is passed on and its element type (as _logits)."""
    if a is None:
        raise NullPointerError(name)
    return _logits(a)


def norm(x, weight=None, *, bias=None, kind: int = NORM_RMS, eps: float = 1e-6, post_weight=None, gate=None,
         scale: float = 1.0, residual=None, hidden_type: int | None = None, y_type: int = _native.F32):
    """The norms around a block (gollek_hip_norm) on host arrays: x (rows, cols)
    float32, float16 or uint16 bf16 bit patterns, residual likewise (its type is
    hidden's; without one hidden_type, by default x's), vectors (cols,) float32 ->
    hidden, y."""
    xv, x_type = _typed(x, "input")
    if xv.ndim != 2:
        raise IllegalArgumentError("input must be (rows, cols)")
    rows, cols = xv.shape
    rv = None
    if residual is not None:
        rv, r_type = _logits(residual)
        if rv.shape != xv.shape or hidden_type not in (None, r_type):
            raise IllegalArgumentError(f"residual must be {xv.shape} of the hidden type")
        hidden_type = r_type
    hidden_type = x_type if hidden_type is None else hidden_type
    for t in (hidden_type, y_type):
        if t not in _LINEAR_DTYPES:
            raise UnsupportedOperationError(f"Unsupported norm type id: {t} (F32, F16 or BF16)")

    def vector(v, name):
        if v is None:
            return None
        v = np.ascontiguousarray(v, dtype=np.float32)
        if v.shape != (cols,):
            raise IllegalArgumentError(f"{name} must be ({cols},)")
        return v

    vs = [vector(v, n) for v, n in ((post_weight, "post_weight"), (gate, "gate"), (weight, "weight"), (bias, "bias"))]
    at = [None if v is None else v.ctypes.data for v in vs]
    h, y = np.empty(xv.shape, _LINEAR_DTYPES[hidden_type]), np.empty(xv.shape, _LINEAR_DTYPES[y_type])
    err = _native.ErrBuf()
    check(_native.load().gollek_hip_norm(xv.ctypes.data, x_type, rows, cols, at[0], at[1], scale,
                                         None if rv is None else rv.ctypes.data, h.ctypes.data, hidden_type, at[2], at[3],
                                         kind, eps, y.ctypes.data, y_type, err.buf, err.size), err)
    return h, y


def norm_device(x_ptr: int, x_type: int, rows: int, cols: int, *, x_stride: int = 0, post_weight_ptr: int = 0,
                gate_ptr: int = 0, scale: float = 1.0, residual_ptr: int = 0, residual_stride: int = 0,
                hidden_ptr: int = 0, hidden_type: int = _native.F32, hidden_stride: int = 0, weight_ptr: int = 0,
                bias_ptr: int = 0, kind: int = NORM_RMS, eps: float = 1e-6, y_ptr: int = 0, y_type: int = _native.BF16,
                y_stride: int = 0, stream: int = 0) -> None:
    """hidden = residual + scale * gate * (norm of x by post_weight, or x), y = norm
    of that by weight and bias (gollek_hip_norm_device); 0 leaves a part out."""
    err = _native.err_buf()
    check(_native.load().gollek_hip_norm_device(x_ptr, x_type, rows, cols, x_stride, post_weight_ptr, gate_ptr, scale,
                                                residual_ptr, residual_stride, hidden_ptr, hidden_type, hidden_stride,
                                                weight_ptr, bias_ptr, kind, eps, y_ptr, y_type, y_stride, stream,
                                                err.buf, err.size), err)


def _factors(factors, dims):
    if factors is None:
        return None
    f = np.ascontiguousarray(factors, dtype=np.float32)
    if f.shape != (dims // 2,):
        raise IllegalArgumentError(f"factors must be ({dims // 2},)")
    return f


def rope_frequencies(dims: int, *, base: float = 10000.0, scaling: int = ROPE_NONE, factor: float = 1.0,
                     original_context: float = 0.0, low: float = 0.0, high: float = 0.0, magnitude: float = 0.0,
                     factors=None):
    """Radians a position of each pair (dims / 2,) float32 and the magnitude
    (gollek_hip_rope_frequencies; needs no GPU)."""
    f = _factors(factors, dims)
    out, result = np.empty(max(dims, 0) // 2, np.float32), ctypes.c_float()
    err = _native.ErrBuf()
    check(_native.load().gollek_hip_rope_frequencies(dims, base, scaling, factor, original_context, low, high, magnitude,
                                                     None if f is None else f.ctypes.data, out.ctypes.data,
                                                     ctypes.addressof(result), err.buf, err.size), err)
    return out, result.value


class Rope:
    """A model's rotary table on the current device (gollek_hip_rope).  Keep it as long as
    the model: it must outlive its calls and the captured graphs that hold one."""

    def __init__(self, dims: int, *, layout: int = ROPE_HALF, base: float = 10000.0, scaling: int = ROPE_NONE,
                 factor: float = 1.0, original_context: float = 0.0, low: float = 0.0, high: float = 0.0,
                 magnitude: float = 0.0, factors=None):
        f = _factors(factors, dims)
        err = _native.ErrBuf()
        lib = _native.load()
        self.handle = lib.gollek_hip_rope_create(layout, dims, base, scaling, factor, original_context, low, high,
                                                 magnitude, None if f is None else f.ctypes.data, err.buf, err.size)
        if not self.handle:
            check(lib.gollek_hip_last_status(), err)
        self.dims = dims

    def close(self) -> None:
        if self.handle:
            _native.load().gollek_hip_rope_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def apply(self, x, positions) -> np.ndarray:
        """x (tokens, heads, head_dim) float32, float16 or uint16 bf16 bit patterns,
        rotated to positions (tokens,)."""
        xv, kind = _typed(x, "input")
        if positions is None:
            raise NullPointerError("positions")
        pv = np.ascontiguousarray(positions, dtype=np.int32)
        if xv.ndim != 3 or pv.shape != xv.shape[:1]:
            raise IllegalArgumentError("input must be (tokens, heads, head_dim) and positions (tokens,)")
        out = np.empty_like(xv)
        err = _native.ErrBuf()
        check(_native.load().gollek_hip_rope_apply(self.handle, xv.ctypes.data, kind, *xv.shape, pv.ctypes.data,
                                                   out.ctypes.data, err.buf, err.size), err)
        return out

    def apply_device(self, x_ptr: int, type_id: int, tokens: int, heads: int, head_dim: int, positions_ptr: int,
                     out_ptr: int, *, x_stride: int = 0, out_stride: int = 0, stream: int = 0) -> None:
        err = _native.err_buf()
        check(_native.load().gollek_hip_rope_apply_device(self.handle, x_ptr, type_id, tokens, heads, head_dim, x_stride,
                                                          positions_ptr, out_ptr, out_stride, stream, err.buf,
                                                          err.size), err)


class KvCache:
    """A paged cache of keys and values in the caller's device memory
    (gollek_hip_kv_cache): k and v (pages, kv_heads, page_size, head_dim) of F16 or
    BF16, which must outlive it and the captured graphs that hold a call on it."""

    def __init__(self, type_id: int, k_ptr: int, v_ptr: int, pages: int, page_size: int, kv_heads: int, head_dim: int):
        err = _native.ErrBuf()
        lib = _native.load()
        self.handle = lib.gollek_hip_kv_cache_wrap_device(type_id, k_ptr, v_ptr, pages, page_size, kv_heads, head_dim,
                                                          err.buf, err.size)
        if not self.handle:
            check(lib.gollek_hip_last_status(), err)

    def close(self) -> None:
        if self.handle:
            _native.load().gollek_hip_kv_cache_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def append(self, k_ptr: int, v_ptr: int, type_id: int, tokens: int, positions_ptr: int, page_table_ptr: int,
               sequences: int, max_pages: int, *, rope: Rope | None = None, k_stride: int = 0, v_stride: int = 0,
               q_ptr: int = 0, q_heads: int = 0, q_stride: int = 0, q_out_ptr: int = 0, q_out_stride: int = 0,
               q_norm_ptr: int = 0, k_norm_ptr: int = 0, eps: float = 1e-6, sequence_ptr: int = 0,
               stream: int = 0) -> None:
        """New tokens' keys (normalised, rotated) and values into their pages, their
        queries (normalised, rotated) to q_out (gollek_hip_kv_append_device)."""
        if rope is not None and not rope.handle:
            raise NullPointerError("rotary table")  # a closed one: not the call without rotation
        err = _native.err_buf()
        check(_native.load().gollek_hip_kv_append_device(
            self.handle, None if rope is None else rope.handle, k_ptr, k_stride, v_ptr, v_stride, q_ptr, q_heads,
            q_stride, type_id, tokens, q_norm_ptr, k_norm_ptr, eps, positions_ptr, sequence_ptr, page_table_ptr,
            sequences, max_pages, q_out_ptr, q_out_stride, stream, err.buf, err.size), err)

    def attend_workspace_bytes(self, sequences: int, q_heads: int, max_pages: int) -> int:
        return int(_native.load().gollek_hip_attention_workspace_bytes(self.handle, sequences, q_heads, max_pages))

    def attend(self, q_ptr: int, sequences: int, q_heads: int, lengths_ptr: int, page_table_ptr: int, max_pages: int,
               out_ptr: int, out_type: int, *, scale: float, softcap: float = 0.0, window: int = 0, sinks_ptr: int = 0,
               q_stride: int = 0, out_stride: int = 0, ws_ptr: int = 0, ws_bytes: int = 0, stream: int = 0) -> None:
        """Attention of one new token a sequence over the first lengths of its pages
        (gollek_hip_attention_device)."""
        err = _native.err_buf()
        check(_native.load().gollek_hip_attention_device(
            self.handle, q_ptr, q_stride, sequences, q_heads, lengths_ptr, page_table_ptr, max_pages, scale, softcap,
            window, sinks_ptr, out_ptr, out_type, out_stride, ws_ptr, ws_bytes, stream, err.buf, err.size), err)
