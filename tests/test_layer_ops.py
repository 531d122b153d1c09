"""CPU tests of norms, rotary positions, the paged cache and its attention: what is
refused before any device call, and the rotary tables' frequencies."""
import ctypes
import math

import numpy as np
import pytest

from gollek_amd import _native
from gollek_amd import tensor_ops as ops

F32, F16, BF16 = _native.F32, _native.F16, _native.BF16
BASE = 1 << 20  # addresses that no call here reaches


def norm_device(**kw):
    call = dict(x_ptr=BASE, x_type=BF16, rows=4, cols=64, hidden_ptr=BASE + 65536, hidden_type=F32, y_ptr=BASE + 131072,
                y_type=BF16)
    call.update(kw)
    ops.norm_device(**call)


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=1 << 31), dict(cols=0), dict(cols=65537), dict(kind=2), dict(scale=float("inf")),
    dict(scale=float("nan")), dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(x_stride=63),
    dict(y_stride=63), dict(hidden_stride=-64), dict(x_ptr=BASE + 1), dict(y_ptr=BASE + 131073),
    dict(hidden_ptr=BASE + 65538), dict(weight_ptr=BASE + 300001), dict(x_stride=1 << 60),
    dict(y_ptr=BASE + 64, x_stride=128, y_stride=128),              # y over half of x's rows
    dict(y_ptr=BASE, y_type=F32),                                   # wider than what it lies on
    dict(y_ptr=BASE, y_stride=128),                                 # another pitch
    dict(y_ptr=BASE + 65536, y_type=F32),                           # hidden
    dict(residual_ptr=BASE + 65536 + 4),                            # hidden one element off its residual
    dict(weight_ptr=BASE + 131072 + 128), dict(gate_ptr=BASE + 65536), dict(bias_ptr=BASE + 131072),
    dict(post_weight_ptr=BASE + 65536 + 64)])
def test_norm_refuses(kw):
    with pytest.raises(ops.IllegalArgumentError):
        norm_device(**kw)


@pytest.mark.parametrize("kw", [dict(x_ptr=0), dict(hidden_ptr=0, y_ptr=0)])
def test_norm_refuses_null(kw):
    with pytest.raises(ops.NullPointerError):
        norm_device(**kw)


@pytest.mark.parametrize("kw", [dict(x_type=2), dict(y_type=8), dict(hidden_type=-1)])
def test_norm_refuses_types(kw):
    with pytest.raises(ops.UnsupportedOperationError):
        norm_device(**kw)


def test_norm_of_no_rows_does_nothing():
    norm_device(rows=0, x_ptr=0, hidden_ptr=0, y_ptr=0)


def test_host_norm_refuses():
    x = np.zeros((2, 8), np.float32)
    with pytest.raises(ops.NullPointerError):
        ops.norm(None)
    with pytest.raises(ops.IllegalArgumentError):
        ops.norm(x[0])
    with pytest.raises(ops.IllegalArgumentError):
        ops.norm(x, np.ones(7))
    with pytest.raises(ops.IllegalArgumentError):
        ops.norm(x, residual=np.zeros((2, 9), np.float32))
    with pytest.raises(ops.IllegalArgumentError):
        ops.norm(x, residual=np.zeros((2, 8), np.float16), hidden_type=F32)
    with pytest.raises(ops.UnsupportedOperationError):
        ops.norm(x, y_type=8)
    with pytest.raises(ops.IllegalArgumentError):
        ops.norm(x, eps=-1.0)


def test_frequencies_unscaled_and_linear():
    f, magnitude = ops.rope_frequencies(64, base=500000.0)
    want = 500000.0 ** (-2.0 * np.arange(32) / 64)
    assert magnitude == 1.0 and np.allclose(f, want, rtol=2.0**-23, atol=0)
    f, magnitude = ops.rope_frequencies(64, base=500000.0, scaling=ops.ROPE_LINEAR, factor=4.0, magnitude=1.5)
    assert magnitude == 1.5 and np.allclose(f, want / 4, rtol=2.0**-23, atol=0)
    factors = np.linspace(1, 8, 32).astype(np.float32)
    f, _ = ops.rope_frequencies(64, base=500000.0, factors=factors)
    assert np.allclose(f, want / factors, rtol=2.0**-23, atol=0)


@pytest.mark.parametrize("dims,base,factor,context", [(128, 10000.0, 16.0, 4096.0), (128, 1000000.0, 4.0, 32768.0),
                                                      (20, 10000.0, 40.0, 4096.0), (2, 10000.0, 8.0, 512.0)])
def test_yarn_frequencies(dims, base, factor, context):
    f, magnitude = ops.rope_frequencies(dims, base=base, scaling=ops.ROPE_YARN, factor=factor, original_context=context,
                                        low=1.0, high=32.0)
    plain = base ** (-2.0 * np.arange(dims // 2) / dims)

    def pair(turns):  # the pair that turns so many times in the context
        return dims * math.log(context / (2 * math.pi * turns)) / (2 * math.log(base))

    lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), dims - 1)
    ramp = np.clip((np.arange(dims // 2) - lo) / max(hi - lo, 0.001), 0, 1)
    assert np.allclose(f, plain * (1 - ramp) + plain / factor * ramp, rtol=2.0**-22, atol=0)
    assert abs(magnitude - (0.1 * math.log(factor) + 1)) < 2.0**-22
    assert np.allclose(f[ramp == 0], plain[ramp == 0], rtol=2.0**-23, atol=0)


def test_llama3_frequencies():
    f, magnitude = ops.rope_frequencies(128, base=500000.0, scaling=ops.ROPE_LLAMA3, factor=8.0, original_context=8192.0,
                                        low=1.0, high=4.0)
    want = []
    for i in range(64):
        a = 500000.0 ** (-2.0 * i / 128)
        wave = 2 * math.pi / a
        if wave > 8192.0 / 1.0:
            a /= 8
        elif wave > 8192.0 / 4.0:
            s = (8192.0 / wave - 1.0) / 3.0
            a = (1 - s) * a / 8 + s * a
        want.append(a)
    assert magnitude == 1.0 and np.allclose(f, want, rtol=2.0**-22, atol=0)


@pytest.mark.parametrize("kw", [
    dict(dims=0), dict(dims=3), dict(dims=258), dict(dims=-2), dict(base=1.0), dict(base=float("nan")),
    dict(base=float("inf")), dict(scaling=4), dict(scaling=-1), dict(scaling=1, factor=0.0),
    dict(scaling=1, factor=float("nan")), dict(magnitude=-1.0), dict(magnitude=float("nan")),
    dict(scaling=2, factor=4.0), dict(scaling=2, factor=4.0, original_context=4096.0, low=32.0, high=1.0),
    dict(scaling=3, factor=8.0, original_context=8192.0, low=0.0, high=4.0),
    dict(scaling=3, factor=8.0, original_context=float("inf"), low=1.0, high=4.0),
    dict(factors=np.zeros(32, np.float32)), dict(factors=np.ones(31, np.float32))])
def test_rope_refuses(kw):
    call = dict(dims=64)
    call.update(kw)
    with pytest.raises(ops.IllegalArgumentError):
        ops.rope_frequencies(**call)
    with pytest.raises(ops.IllegalArgumentError):
        ops.Rope(**call)


def test_rope_refuses_layouts_and_null():
    with pytest.raises(ops.IllegalArgumentError):
        ops.Rope(64, layout=2)
    lib, e = _native.load(), _native.ErrBuf()
    assert lib.gollek_hip_rope_apply_device(None, BASE, F32, 1, 1, 64, 0, BASE, BASE, 0, None, e.buf,
                                            e.size) == _native.ERR_NULL
    assert lib.gollek_hip_rope_apply(None, None, F32, 1, 1, 64, None, None, e.buf, e.size) == _native.ERR_NULL
    lib.gollek_hip_rope_free(None)  # ignored


def cache(**kw):
    call = dict(type_id=BF16, k_ptr=BASE, v_ptr=BASE + (1 << 20), pages=4, page_size=16, kv_heads=2, head_dim=64)
    call.update(kw)
    return ops.KvCache(**call)


@pytest.mark.parametrize("kw", [
    dict(pages=0), dict(pages=1 << 31), dict(page_size=8), dict(page_size=24), dict(page_size=1 << 17), dict(kv_heads=0),
    dict(kv_heads=65536), dict(head_dim=0), dict(head_dim=12), dict(head_dim=264), dict(k_ptr=BASE + 8),
    dict(v_ptr=BASE + 2), dict(v_ptr=BASE + 16), dict(pages=(1 << 31) - 1, page_size=65536, kv_heads=65535, head_dim=256)])
def test_cache_refuses(kw):
    with pytest.raises(ops.IllegalArgumentError):
        cache(**kw)


def test_cache_refuses_types_and_null():
    with pytest.raises(ops.UnsupportedOperationError):
        cache(type_id=F32)
    with pytest.raises(ops.NullPointerError):
        cache(k_ptr=0)
    _native.load().gollek_hip_kv_cache_free(None)  # ignored


def append(c, **kw):
    call = dict(k_ptr=BASE + (4 << 20), v_ptr=BASE + (5 << 20), type_id=F32, tokens=3, positions_ptr=BASE + (6 << 20),
                page_table_ptr=BASE + (7 << 20), sequences=3, max_pages=4, q_ptr=BASE + (8 << 20), q_heads=4,
                q_out_ptr=BASE + (9 << 20))
    call.update(kw)
    c.append(**call)


@pytest.mark.parametrize("kw", [
    dict(tokens=-1), dict(tokens=1 << 31), dict(q_heads=-1), dict(q_heads=65536), dict(sequences=-1), dict(max_pages=0),
    dict(max_pages=1 << 27), dict(eps=-1.0), dict(eps=float("nan")), dict(k_stride=127), dict(q_out_stride=255),
    dict(k_ptr=BASE + (4 << 20) + 2), dict(positions_ptr=BASE + (6 << 20) + 1), dict(q_norm_ptr=BASE + (10 << 20) + 2),
    dict(k_ptr=BASE + 64), dict(v_ptr=BASE + (1 << 20)), dict(q_ptr=BASE), dict(q_out_ptr=BASE + 128),
    dict(q_out_ptr=BASE + (4 << 20)), dict(q_out_ptr=BASE + (6 << 20)), dict(q_out_ptr=BASE + (7 << 20) + 16),
    dict(q_out_ptr=BASE + (8 << 20)),                                          # f32 queries, 16-bit results
    dict(positions_ptr=BASE + 16), dict(page_table_ptr=BASE + (1 << 20) + 64), dict(sequence_ptr=BASE + 4)])
def test_append_refuses(kw):
    c = cache()
    with pytest.raises(ops.IllegalArgumentError):
        append(c, **kw)


@pytest.mark.parametrize("kw", [dict(k_ptr=0), dict(v_ptr=0), dict(positions_ptr=0), dict(page_table_ptr=0),
                                dict(q_ptr=0), dict(q_out_ptr=0)])
def test_append_refuses_null(kw):
    c = cache()
    with pytest.raises(ops.NullPointerError):
        append(c, **kw)
    with pytest.raises(ops.UnsupportedOperationError):
        append(c, type_id=2)


def test_append_refuses_a_closed_table():
    rope = ops.Rope.__new__(ops.Rope)
    rope.handle, rope.dims = None, 64
    with pytest.raises(ops.NullPointerError):
        append(cache(), rope=rope)
    closed = cache()
    closed.close()
    with pytest.raises(ops.NullPointerError):
        append(closed)


def test_append_and_attend_refuse_a_null_cache():
    lib, e = _native.load(), _native.ErrBuf()
    assert lib.gollek_hip_kv_append_device(None, None, None, 0, None, 0, None, 0, 0, F32, 0, None, None, 0.0, None, None,
                                           None, 0, 1, None, 0, None, e.buf, e.size) == _native.ERR_NULL
    assert lib.gollek_hip_attention_device(None, None, 0, 0, 1, None, None, 1, 1.0, 0.0, 0, None, None, F32, 0, None, 0,
                                           None, e.buf, e.size) == _native.ERR_NULL
    assert lib.gollek_hip_attention_workspace_bytes(None, 1, 1, 1) == -1


def attend(c, **kw):
    call = dict(q_ptr=BASE + (4 << 20), sequences=3, q_heads=4, lengths_ptr=BASE + (5 << 20),
                page_table_ptr=BASE + (6 << 20), max_pages=4, out_ptr=BASE + (7 << 20), out_type=F32, scale=0.125,
                ws_ptr=BASE + (64 << 20), ws_bytes=1 << 30)
    call.update(kw)
    c.attend(**call)


@pytest.mark.parametrize("kw", [
    dict(sequences=-1), dict(sequences=65536), dict(q_heads=0), dict(q_heads=3), dict(q_heads=65536),
    dict(sequences=65535, q_heads=512), dict(max_pages=0), dict(max_pages=1 << 27), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")),
    dict(scale=2e15), dict(scale=-1e30), dict(softcap=1e-30), dict(softcap=1e20), dict(window=-1), dict(q_stride=255), dict(out_stride=255), dict(q_ptr=BASE + (4 << 20) + 1),
    dict(out_ptr=BASE + (7 << 20) + 2), dict(lengths_ptr=BASE + (5 << 20) + 2), dict(sinks_ptr=BASE + (8 << 20) + 1),
    dict(out_ptr=BASE + (4 << 20), out_type=BF16), dict(out_ptr=BASE + 256), dict(out_ptr=BASE + (1 << 20)),
    dict(out_ptr=BASE + (5 << 20)), dict(out_ptr=BASE + (6 << 20)), dict(sinks_ptr=BASE + (7 << 20)),
    dict(ws_ptr=BASE + (64 << 20) + 128)])
def test_attend_refuses(kw):
    c = cache()
    with pytest.raises(ops.IllegalArgumentError):
        attend(c, **kw)


@pytest.mark.parametrize("kw", [dict(q_ptr=0), dict(out_ptr=0), dict(lengths_ptr=0), dict(page_table_ptr=0)])
def test_attend_refuses_null(kw):
    c = cache()
    with pytest.raises(ops.NullPointerError):
        attend(c, **kw)
    with pytest.raises(ops.UnsupportedOperationError):
        attend(c, out_type=2)


def test_attend_workspace():
    c = cache()
    need = c.attend_workspace_bytes(3, 4, 4096)
    assert need >= 0
    if need:
        with pytest.raises(ops.IllegalArgumentError):
            attend(c, max_pages=4096, ws_bytes=need - 1)
        with pytest.raises(ops.NullPointerError):
            attend(c, max_pages=4096, ws_ptr=0)
        with pytest.raises(ops.IllegalArgumentError):  # the workspace over the queries
            attend(c, max_pages=4096, ws_ptr=BASE + (4 << 20))
    sizes = [c.attend_workspace_bytes(n, 4, p) for n in (0, 1, 2, 7, 64, 300, 5000) for p in (4096,)]
    assert sizes[0] == 0 and sizes == sorted(sizes)
    for n in (1, 8, 400):
        sizes = [c.attend_workspace_bytes(n, 4, p) for p in (1, 2, 9, 64, 1000, 100000)]
        assert sizes == sorted(sizes)
    for dim in (8, 64, 128, 192, 256):
        for page in (16, 64):
            c = cache(head_dim=dim, page_size=page, v_ptr=BASE + (1 << 24), kv_heads=8)
            table = [[c.attend_workspace_bytes(n, 16, p) for p in (1, 3, 5, 8, 15, 23, 25, 33, 49, 70, 97, 130, 500, 9000)]
                     for n in (1, 2, 3, 5, 6, 9, 31, 32, 33, 64, 127, 256, 1023, 1024, 1025, 3000, 65535)]
            assert all(row == sorted(row) for row in table) and all(list(col) == sorted(col) for col in zip(*table))
    c = cache()
    assert c.attend_workspace_bytes(1, 3, 4) == -1 and c.attend_workspace_bytes(65536, 4, 4) == -1


def test_calls_of_no_rows_do_nothing():
    c = cache()
    append(c, tokens=0, k_ptr=0, v_ptr=0, q_ptr=0, q_out_ptr=0, positions_ptr=0, page_table_ptr=0)
    attend(c, sequences=0, q_ptr=0, out_ptr=0, lengths_ptr=0, page_table_ptr=0, ws_ptr=0, ws_bytes=0)


def test_status_and_message_of_a_refusal():
    lib, e = _native.load(), _native.ErrBuf()
    assert lib.gollek_hip_rope_frequencies(3, 10000.0, 0, 1.0, 0.0, 0.0, 0.0, 0.0, None, None, None, e.buf,
                                           e.size) == _native.ERR_ARG
    assert "rotary dimensions" in e.text and lib.gollek_hip_last_status() == _native.ERR_ARG
    small = ctypes.create_string_buffer(8)
    lib.gollek_hip_rope_frequencies(3, 10000.0, 0, 1.0, 0.0, 0.0, 0.0, 0.0, None, None, None, small, 8)
    assert len(small.value) == 7
