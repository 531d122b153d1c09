"""CPU tests of the C-ABI library: it loads, exports every symbol its header
declares, and rejects bad arguments before touching a device, with the status
codes the Java adapter maps back to the reference's exceptions."""
import ctypes
import re
from pathlib import Path

import numpy as np
import pytest

from gollek_amd import _native
from gollek_amd import tensor_ops as ops

HEADER = Path(__file__).resolve().parents[1] / "include" / "gollek_hip.h"


def declared_functions() -> list[str]:
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(gollek_hip_\w+)\s*\(", text)))


def test_library_exports_every_declared_symbol():
    lib = _native.load()
    names = declared_functions()
    assert len(names) >= 12
    missing = [n for n in names if not hasattr(lib, n)]
    assert not missing, missing


def test_library_resolves_all_of_its_own_symbols():
    # Loading binds lazily here, so an unresolved kernel launch stub (which
    # hipcc can leave behind for a kernel template) would only fail on first
    # use; dlopen with RTLD_NOW resolves every symbol up front.
    lib_path = _native.load()._name
    ctypes.CDLL(lib_path, mode=ctypes.RTLD_GLOBAL | 0x2)  # RTLD_NOW


def test_python_signatures_cover_header():
    assert set(declared_functions()) <= set(_native.SIGNATURES)


def test_version():
    assert _native.load().gollek_hip_version() >= 10000


def _err():
    return _native.ErrBuf()


def test_upload_rejects_unsupported_type():
    lib = _native.load()
    e = _err()
    buf = np.zeros(64, np.uint8)
    h = lib.gollek_hip_weight_upload(1, buf.ctypes.data, 1, 32, 64, e.buf, e.size)  # F16
    assert not h
    assert lib.gollek_hip_last_status() == _native.ERR_UNSUPPORTED
    assert "Unsupported" in e.text


def test_upload_rejects_non_block_multiple():
    lib = _native.load()
    e = _err()
    buf = np.zeros(1024, np.uint8)
    h = lib.gollek_hip_weight_upload(_native.Q4_K, buf.ctypes.data, 1, 300, 144, e.buf, e.size)
    assert not h
    assert lib.gollek_hip_last_status() == _native.ERR_ARG
    assert "not a multiple of block size 256" in e.text


def test_upload_rejects_wrong_row_bytes_and_null():
    lib = _native.load()
    e = _err()
    buf = np.zeros(1024, np.uint8)
    assert not lib.gollek_hip_weight_upload(_native.Q8_0, buf.ctypes.data, 2, 64, 70, e.buf, e.size)
    assert lib.gollek_hip_last_status() == _native.ERR_ARG
    assert not lib.gollek_hip_weight_upload(_native.Q8_0, None, 2, 64, 68, e.buf, e.size)
    assert lib.gollek_hip_last_status() == _native.ERR_NULL


def test_null_handle_calls_fail_with_null_status():
    lib = _native.load()
    e = _err()
    x = np.zeros(32, np.float32)
    y = np.zeros(4, np.float32)
    assert lib.gollek_hip_matvec_rows(None, x.ctypes.data, 32, y.ctypes.data, 4, 1, e.buf,
                                      e.size) == _native.ERR_NULL
    assert lib.gollek_hip_dot_row(None, 0, x.ctypes.data, 32, y.ctypes.data, e.buf,
                                  e.size) == _native.ERR_NULL
    assert lib.gollek_hip_dequantize_rows(None, 0, 1, y.ctypes.data, 4, e.buf,
                                          e.size) == _native.ERR_NULL
    assert lib.gollek_hip_matvec_device(None, None, None, 0, None, e.buf, e.size) == _native.ERR_NULL
    assert lib.gollek_hip_weight_info(None, None, None, None, None) == _native.ERR_NULL
    lib.gollek_hip_weight_free(None)  # ignored


def test_error_buffer_truncates():
    lib = _native.load()
    small = ctypes.create_string_buffer(8)
    buf = np.zeros(64, np.uint8)
    assert not lib.gollek_hip_weight_upload(99, buf.ctypes.data, 1, 32, 34, small, 8)
    assert len(small.value) == 7


def test_testing_option_is_outside_the_public_abi():
    # The kernel-family switch the parity tests use is exported by a
    # test-only header, not by include/gollek_hip.h.
    assert "gollek_hip_testing_set_option" not in declared_functions()
    assert "gollek_hip_set_option" not in declared_functions()
    ops.set_option("gemv_variant", 0)
    with pytest.raises(ops.IllegalArgumentError):
        ops.set_option("no_such_option", 1)
    with pytest.raises(ops.IllegalArgumentError):
        ops.set_option("gemv_variant", 2)


def test_tensor_shape_rules():
    t = ops.GgufTensor("blk.0.ffn_up.weight", (4096, 11008), 2, np.zeros(1, np.uint8))
    assert (t.columns, t.rows, t.row_bytes) == (4096, 11008, 2304)
    t = ops.GgufTensor("ffn_gate_exps", (2048, 768, 128), 12, np.zeros(1, np.uint8))
    assert (t.columns, t.rows, t.row_bytes) == (2048, 768 * 128, 1152)


def test_python_mirror_null_checks():
    with pytest.raises(ops.NullPointerError):
        ops.mat_vec_rows(None, np.zeros(4, np.float32), np.zeros(4, np.float32), 1)
    with pytest.raises(ops.NullPointerError):
        ops.dot_row(None, 0, np.zeros(4, np.float32))


def test_linear_refuses_a_null_weight():
    lib = _native.load()
    e = _err()
    x, y = np.zeros(32, np.uint16), np.zeros(4, np.float32)
    assert lib.gollek_hip_linear(None, x.ctypes.data, 32, 1, None, 0, None, None, y.ctypes.data, _native.F32, 4, e.buf,
                                 e.size) == _native.ERR_NULL
    assert lib.gollek_hip_linear_device(None, None, 1, None, 0, None, 0, None, 0, None, _native.F32, 0, None, 0, None,
                                        e.buf, e.size) == _native.ERR_NULL
    assert lib.gollek_hip_linear_workspace_bytes(None, 1) == -1
    with pytest.raises(ops.NullPointerError):
        ops.linear(None, np.zeros((1, 32), np.uint16))


@pytest.mark.parametrize("kw", [dict(n_groups=5), dict(n_groups=0), dict(n_groups=2, top_groups=3), dict(top_groups=0),
                                dict(group_top=0), dict(group_top=3), dict(top_k=33), dict(top_k=0),
                                dict(n_groups=4, top_groups=1, top_k=9), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(scoring=2), dict(bias=np.zeros(31, np.float32))])
def test_route_refuses(kw):
    call = dict(top_k=4, scoring=0)
    call.update(kw)
    with pytest.raises(ops.IllegalArgumentError):
        ops.moe_route(np.zeros((3, 32), np.float32), **call)


def test_route_refuses_types_nulls_and_misaligned_logits():
    lib, e = _native.load(), _err()

    def rc(logits=4096, kind=0, tokens=1, experts=32, bias=0, ids=4096, w=4096):
        return lib.gollek_hip_moe_route_device(logits, kind, tokens, experts, bias, 0, 1, 1, 1, 2, 1, 1.0, ids, w, None,
                                               e.buf, e.size)

    assert rc(kind=8) == _native.ERR_UNSUPPORTED
    assert rc(logits=0) == rc(ids=0) == rc(w=0) == _native.ERR_NULL
    assert rc(logits=4098) == rc(logits=4097, kind=30) == rc(bias=4098) == _native.ERR_ARG
    assert rc(tokens=-1) == rc(experts=4097) == rc(experts=0) == _native.ERR_ARG
    assert rc(tokens=0, logits=0) == _native.OK
    with pytest.raises(ops.NullPointerError):
        ops.moe_route(None, 2, 0)
    with pytest.raises(ops.IllegalArgumentError):
        ops.moe_route(np.zeros(32, np.float32), 2, 0)


def test_sample_refuses():
    lib, e = _native.load(), _err()

    def rc(logits=4096, kind=0, rows=1, vocab=100, stride=0, t=0, k=0, p=0, mp=0, u=4096, tok=4096, prob=0, kept=0,
           ws=256, ws_bytes=1 << 40):
        return lib.gollek_hip_sample_device(logits, kind, rows, vocab, stride, t, k, p, mp, u, tok, prob, kept, ws,
                                            ws_bytes, None, e.buf, e.size)

    assert rc(kind=8) == _native.ERR_UNSUPPORTED
    assert rc(logits=0) == rc(u=0) == rc(tok=0) == _native.ERR_NULL
    for bad in (dict(rows=-1), dict(rows=65536), dict(vocab=0), dict(vocab=(1 << 22) + 1), dict(stride=99),
                dict(stride=-1), dict(logits=4098), dict(logits=4097, kind=1), dict(t=4098), dict(k=4097), dict(p=4098),
                dict(mp=4098), dict(u=4098), dict(tok=4098), dict(prob=4098), dict(kept=4098), dict(ws=128)):
        assert rc(**bad) == _native.ERR_ARG, bad
    assert rc(rows=0, logits=0, u=0, tok=0) == _native.OK
    assert lib.gollek_hip_sample_workspace_bytes(1, 0) == lib.gollek_hip_sample_workspace_bytes(-1, 10) == -1
    need = lib.gollek_hip_sample_workspace_bytes(1, 100)
    if need > 0:
        assert rc(ws=0) == _native.ERR_NULL and rc(ws_bytes=need - 1) == _native.ERR_ARG
    l, u = np.zeros((2, 8), np.float32), np.zeros(2, np.float32)
    for kw in (dict(top_k=[1, 2, 3]), dict(temperature=np.zeros((2, 1)))):
        with pytest.raises(ops.IllegalArgumentError):
            ops.sample(l, u, **kw)
    with pytest.raises(ops.IllegalArgumentError):
        ops.sample(l[0], u)
    for a in ((None, u), (l, None)):
        with pytest.raises(ops.NullPointerError):
            ops.sample(*a)
    with pytest.raises(ops.NullPointerError):
        ops.next_token(None, u, 0.5)
    assert lib.gollek_hip_next_token(None, u.ctypes.data, 2, 1.0, 0, 1.0, 0.0, 0.5, u.ctypes.data, None, None, e.buf,
                                     e.size) == _native.ERR_NULL


def test_sample_checks_the_workspace_of_long_rows():
    lib, e = _native.load(), _err()
    need = lib.gollek_hip_sample_workspace_bytes(3, 100000)
    assert need > 0 and need % 256 == 0

    def rc(ws, ws_bytes):
        return lib.gollek_hip_sample_device(4096, 0, 3, 100000, 0, 0, 0, 0, 0, 4096, 4096, 0, 0, ws, ws_bytes, None,
                                            e.buf, e.size)

    assert rc(0, need) == _native.ERR_NULL
    assert rc(4096, need - 1) == rc(4096 + 128, need) == _native.ERR_ARG


def test_route_refuses_misaligned_results():
    lib, e = _native.load(), _err()
    for ids, w in ((4098, 4096), (4096, 4097)):
        assert lib.gollek_hip_moe_route_device(4096, 0, 1, 32, 0, 0, 1, 1, 1, 2, 1, 1.0, ids, w, None, e.buf,
                                               e.size) == _native.ERR_ARG


@pytest.mark.parametrize("dtype,kind", [(np.float32, _native.F32), (np.float64, _native.F32), (np.float16, _native.F16),
                                        (np.uint16, _native.BF16)])
def test_logits_go_on_as_what_they_are(monkeypatch, dtype, kind):
    """uint16 logits are bf16 bit patterns, as linear returns them, not numbers."""
    calls = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: calls.append((name, a)) or _native.OK

    monkeypatch.setattr(_native, "load", Library)
    values = np.array([[1, 0x4000, 0x3F80, 7]], dtype)
    ops.sample(values, [0.5])
    ops.moe_route(values, 2, ops.ROUTER_SOFTMAX)
    assert [name for name, _ in calls] == ["gollek_hip_sample", "gollek_hip_moe_route"]
    assert [a[1] for _, a in calls] == [kind, kind]


def test_next_token_takes_bf16_bit_patterns(monkeypatch):
    seen = []

    class Library:
        def gollek_hip_next_token(self, handle, x, n, *rest):
            seen.append(list((ctypes.c_float * n).from_address(x)))
            return _native.OK

    class Head:
        def handle(self):
            return None

    monkeypatch.setattr(_native, "load", Library)
    ops.next_token(Head(), np.array([0x3F80, 0xC000, 0, 0x3E20], np.uint16), 0.5)
    ops.next_token(Head(), [1, 2.5], 0.5)
    assert seen == [[1.0, -2.0, 0.0, 0.15625], [1.0, 2.5]]


def test_sample_workspace_never_shrinks():
    """A workspace for the largest batch and vocabulary serves every smaller one."""
    size = _native.load().gollek_hip_sample_workspace_bytes
    for vocab in (1, 16384, 16385, 32000, 128256, 262145, 4194304):
        rows = list(range(0, 2200)) + [4095, 4096, 4097, 30000, 65535]
        sizes = [size(r, vocab) for r in rows]
        assert sizes == sorted(sizes) and sizes[0] >= 0, vocab
    for rows in (1, 2, 31, 32, 33, 96, 1025, 65535):
        sizes = [size(rows, v) for v in (1, 5000, 16384, 16385, 20480, 20481, 50257, 128256, 131072, 131073, 262144,
                                         262145, 1 << 20, 1 << 22)]
        assert sizes == sorted(sizes), rows


def test_host_forms_without_a_weight_ask_for_the_device_first():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    lib, e = _native.load(), _err()
    x, out = np.zeros(64, np.float32), np.zeros(64, np.float32)
    xp, op = x.ctypes.data, out.ctypes.data
    calls = {
        "select_topk": lambda: lib.gollek_hip_moe_select_topk(xp, 2, 8, 2, 0, op, op + 64, e.buf, e.size),
        "route": lambda: lib.gollek_hip_moe_route(xp, 0, 2, 8, None, 0, 1, 1, 1, 2, 1, 1.0, op, op + 64, e.buf, e.size),
        "sample": lambda: lib.gollek_hip_sample(xp, 0, 2, 8, None, None, None, None, xp, op, None, None, e.buf, e.size),
    }
    for name, call in calls.items():
        assert call() == _native.ERR_DEVICE, name
        assert b"hipGetDevice failed" in e.buf.value or b"hipSetDevice failed" in e.buf.value, (name, e.buf.value)


def _no_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: only where nothing can be launched")


def test_route_refuses_routes_over_what_it_reads():
    _no_device()
    lib, e = _native.load(), _err()
    t, n, k = 10, 32, 2

    def rc(ids, w, bias=0, kind=0):
        return lib.gollek_hip_moe_route_device(1 << 20, kind, t, n, bias, 0, 1, 1, 1, k, 1, 1.0, ids, w, None, e.buf, e.size)

    free, end, r = 1 << 21, (1 << 20) + 4 * t * n, 4 * t * k
    for over in (1 << 20, (1 << 20) + 4 - r, end - 4):
        assert rc(over, free) == rc(free, over) == _native.ERR_ARG
    assert rc(free, free) == rc(free, free + r - 4) == rc(free + r - 4, free) == _native.ERR_ARG
    assert rc(free, free + r, bias=free - 4 * n + 4) == rc(free, free + 8 * r, bias=free + 9 * r - 4) == _native.ERR_ARG
    # side by side they may stand: these calls end at the device that is not there
    for call in (lambda: rc((1 << 20) - r, end), lambda: rc(end, end + r, bias=end + 2 * r),
                 lambda: rc((1 << 20) + 2 * t * n, free, kind=30)):
        assert call() == _native.ERR_DEVICE


@pytest.mark.parametrize("vocab", [100, 20000])
def test_sample_refuses_results_over_what_it_reads(vocab):
    _no_device()
    lib, e = _native.load(), _err()
    rows, stride = 6, vocab + 12  # gaps of 48 bytes; the results are 24 bytes each
    need = lib.gollek_hip_sample_workspace_bytes(rows, vocab)
    l0, u, ws, free, n = 1 << 20, 1 << 30, 1 << 31, 1 << 33, 4 * rows
    end = l0 + 4 * ((rows - 1) * stride + vocab)

    def rc(tok=free, prob=0, kept=0, ws=ws, t=0, k=0):
        return lib.gollek_hip_sample_device(l0, 0, rows, vocab, stride, t, k, 0, 0, u, tok, prob, kept, ws, 1 << 40, None,
                                            e.buf, e.size)

    gap = l0 + 4 * vocab  # behind the first row
    for over in (l0, l0 + 4 - n, end - 4, gap - 4, gap + 28, l0 + 4 * stride):
        assert rc(tok=over) == rc(prob=over) == rc(kept=over) == _native.ERR_ARG, over - l0
    for over in (u + 4, u - n + 4, free, free + n - 4):
        assert rc(prob=over) == rc(kept=over) == _native.ERR_ARG
    assert rc(tok=u + 4) == rc(k=free + 4) == rc(prob=free + n, kept=free + 2 * n - 4) == _native.ERR_ARG
    if need > 0:
        base = (end + 255) // 256 * 256
        for at in (l0, base - need // 256 * 256, base - 256):
            assert rc(ws=at) == _native.ERR_ARG
        assert rc(tok=ws) == rc(kept=ws + need - 4) == rc(t=ws + 256) == _native.ERR_ARG
        assert rc(ws=u) == rc(ws=u - 256) == _native.ERR_ARG
    # side by side, in a gap between rows, in a setting's own place: these end at the device that is not there
    for kw in (dict(tok=gap, prob=gap + n), dict(tok=l0 - n, prob=end, kept=end + n), dict(tok=u), dict(prob=u, t=u),
               dict(k=free, tok=free), dict(ws=(end + 255) // 256 * 256), dict(tok=ws + need)):
        assert rc(**kw) == _native.ERR_DEVICE, kw
