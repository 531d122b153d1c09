"""The linear layer (product + epilogue) against float64.

Bounds, per output element.  The product: x as the mat-vec kernels hold it is
off by at most 2^-22 of a superblock's largest |x| (22-bit integers; the GEMM
kernels hold it exactly or better), so the sum by 2^-22 max|x| sum|w|; the sum
in fp32 passes at most 32 additions in a matrix instruction, K / 32 in the
accumulators and 32 more over waves and splits, each off by 2^-24 of the sum of
the terms' magnitudes.  A K-quant term is code part minus min part, whose
magnitudes add up to at most 3 max|w| |x| where a code 0 occurs.  The
activations' slopes are at most 1.13, their own fp32 error and the three
epilogue operations' at most 16 roundings of 2^-24.  Last the one rounding to the output
type: half a step, torch.finfo(t).eps / 2 (and half of fp16's smallest
subnormal, 2^-25).
"""
import ctypes

import numpy as np
import pytest
import torch
from scipy.special import erf

from gollek_amd import _native
from gollek_amd import synthetic as syn
from gollek_amd import tensor_ops as ops
from oracle import oracle as o

pytestmark = pytest.mark.gpu

TYPES = {"q4_0": syn.Q4_0, "q8_0": syn.Q8_0, "q4_k": syn.Q4_K, "q5_k": syn.Q5_K, "q6_k": syn.Q6_K}
DTYPE = {_native.F32: torch.float32, _native.F16: torch.float16, _native.BF16: torch.bfloat16}
HALF_STEP = {_native.F32: 2.0**-24, _native.F16: 2.0**-11, _native.BF16: 2.0**-8}


@pytest.fixture(scope="module", autouse=True)
def _init():
    ops.init(0)


def stream():
    return torch.cuda.current_stream().cuda_stream


def activate(act, v):
    if act == ops.ACT_RELU:
        return np.where(v < 0, 0.0, v)
    if act == ops.ACT_SILU:
        with np.errstate(over="ignore"):  # exp(-v) = inf gives the limit, -0
            return v / (1.0 + np.exp(-v))
    if act == ops.ACT_GELU:
        return 0.5 * v * (1.0 + erf(v / np.sqrt(2.0)))
    if act == ops.ACT_GELU_TANH:
        return 0.5 * v * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (v + 0.044715 * v**3)))
    return v


class Weight:
    def __init__(self, type_id, rows, cols, seed):
        self.type_id, self.rows, self.cols = type_id, rows, cols
        self.data = syn.matrix(type_id, rows, cols, seed=seed)
        self.dev = torch.from_numpy(self.data.reshape(-1)).cuda()
        self.handle = ops.DeviceWeight(type_id, self.dev.data_ptr(), rows, cols)
        self.w = o.dequantize(type_id, self.data, cols).astype(np.float64).reshape(rows, cols)

    def workspace(self, m):
        return torch.zeros(max(self.handle.linear_workspace_bytes(m), 256), device="cuda", dtype=torch.uint8)


def operands(m, rows, y_type, seed, bias, mul, residual):
    rng = np.random.default_rng(seed)
    dt = DTYPE[y_type]
    b = torch.from_numpy(rng.normal(size=rows).astype(np.float32)).cuda() if bias else None
    mu = torch.from_numpy(rng.normal(size=(m, rows)).astype(np.float32)).to(dt).cuda() if mul else None
    re = torch.from_numpy(rng.normal(size=(m, rows)).astype(np.float32)).to(dt).cuda() if residual else None
    return b, mu, re


def f64(t):
    return None if t is None else t.double().cpu().numpy()


def expected(wt, xb, act, b, mu, re, y_type):
    """(y, bound) in float64."""
    x = (np.asarray(xb, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    k = wt.cols
    v = x @ wt.w.T
    wabs, wmax = np.abs(wt.w).sum(1), np.abs(wt.w).max(1)
    tol = 2.0**-22 * np.abs(x).max(1)[:, None] * wabs[None, :]
    tol = tol + (64 + k / 32) * 2.0**-24 * np.abs(x).sum(1)[:, None] * 3.0 * wmax[None, :]
    size = np.abs(v)
    if b is not None:
        v = v + f64(b)
        size = size + np.abs(f64(b))
    v, tol = activate(act, v), 1.13 * tol
    if mu is not None:
        v, tol, size = v * f64(mu), tol * np.abs(f64(mu)), size * np.abs(f64(mu))
    if re is not None:
        v, size = v + f64(re), size + np.abs(f64(re))
    tol = tol + 16 * 2.0**-24 * size
    return v, tol + HALF_STEP[y_type] * (np.abs(v) + tol) + (2.0**-25 if y_type == _native.F16 else 0.0)


def check(got, exp, what):
    want, tol = exp
    err = np.abs(f64(got) - want)
    # (a row of zero weights has a bound of 0)
    worst = float(np.divide(err, tol, out=np.where(err > 0, np.inf, 0.0), where=tol > 0).max()) if err.size else 0.0
    print(f"[gpu] {what}: largest error {worst:.3f} of its bound", flush=True)
    assert np.isfinite(f64(got)).all(), what
    assert worst <= 1.0, what


def call(wt, x, m, y, y_type, act=0, b=None, mu=None, re=None, ws=None, **more):
    wt.handle.linear(x.data_ptr(), m, y.data_ptr(), y_type, bias_ptr=0 if b is None else b.data_ptr(), activation=act,
                     mul_ptr=0 if mu is None else mu.data_ptr(), residual_ptr=0 if re is None else re.data_ptr(),
                     ws_ptr=0 if ws is None else ws.data_ptr(), ws_bytes=0 if ws is None else ws.numel(),
                     stream=more.pop("stream", stream()), **more)


# (type, rows, cols, m): one token to prompts, odd row counts, K of one block,
# K that splits, tiles' edges, K that is no multiple of 64 or 256 (Q8_0, Q4_0).
SHAPES = [(t, r, c, m) for t in ("q4_k", "q5_k", "q6_k", "q8_0", "q4_0")
          for r, c, m in ((256, 512, 1), (300, 512, 2), (33, 256, 3), (512, 1024, 4), (100, 2048, 5), (37, 512, 17),
                          (256, 4096, 33), (260, 1024, 130))]
SHAPES += [("q4_k", 512, 8192, 1), ("q5_k", 512, 8192, 2), ("q8_0", 320, 8192, 1), ("q4_0", 320, 4352, 2),
           ("q8_0", 64, 32, 1), ("q8_0", 65, 96, 7), ("q4_0", 70, 160, 40), ("q8_0", 128, 2080, 150),
           ("q4_0", 1, 256, 1), ("q6_k", 1, 256, 9), ("q4_k", 1000, 4096, 64), ("q6_k", 1024, 8192, 5)]


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_linear_matches_float64(i):
    t, rows, cols, m = SHAPES[i]
    act, y_type = i % 5, (_native.F32, _native.BF16, _native.F16)[i % 3]
    bias, mul, residual = i % 2 == 0, i % 4 < 2, i % 3 != 1
    print(f"[gpu] linear {t} {rows}x{cols} m={m} act={act} type={y_type}", flush=True)
    wt = Weight(TYPES[t], rows, cols, 100 + i)
    xb = syn.activation_bf16(m, cols, seed=i)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    b, mu, re = operands(m, rows, y_type, i, bias, mul, residual)
    y = torch.full((m, rows), float("nan"), device="cuda", dtype=DTYPE[y_type])
    call(wt, x, m, y, y_type, act, b, mu, re, wt.workspace(m))
    check(y, expected(wt, xb, act, b, mu, re, y_type), f"{t} {rows}x{cols} m={m}")


@pytest.mark.parametrize("y_type", [_native.F32, _native.F16, _native.BF16])
@pytest.mark.parametrize("act", range(5))
def test_every_activation_in_every_type(act, y_type):
    m, rows, cols = 20, 96, 512
    wt = Weight(syn.Q4_K, rows, cols, 5)
    xb = syn.activation_bf16(m, cols, seed=act)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    b, mu, re = operands(m, rows, y_type, act, True, True, True)
    y = torch.empty((m, rows), device="cuda", dtype=DTYPE[y_type])
    call(wt, x, m, y, y_type, act, b, mu, re, wt.workspace(m))
    check(y, expected(wt, xb, act, b, mu, re, y_type), f"act {act} type {y_type}")


@pytest.mark.parametrize("t,rows,cols,m", [("q4_k", 260, 512, 1), ("q8_0", 260, 512, 24), ("q6_k", 131, 512, 70),
                                           ("q8_0", 512, 4096, 300), ("q4_k", 256, 4096, 48)])
def test_strided_rows_leave_the_rest_alone(t, rows, cols, m):
    wt = Weight(TYPES[t], rows, cols, 6)
    xb = syn.activation_bf16(m, cols, seed=3)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    y_type = _native.BF16
    b, mu, re = operands(m, rows, y_type, 9, True, True, True)
    wide = torch.full((m, 2 * rows + 24), 7.0, device="cuda", dtype=torch.bfloat16)
    wide[:, rows + 13:2 * rows + 13] = mu  # mul in another column range of y's own matrix
    res = torch.zeros((m, rows + 5), device="cuda", dtype=torch.bfloat16)
    res[:, :rows] = re
    before = wide.clone()
    call(wt, x, m, wide[:, 5:], y_type, ops.ACT_SILU, b, wide[:, rows + 13:], res, wt.workspace(m),
         y_stride=wide.shape[1], mul_stride=wide.shape[1], residual_stride=res.shape[1])
    check(wide[:, 5:5 + rows], expected(wt, xb, ops.ACT_SILU, b, mu, re, y_type), "strided")
    assert torch.equal(wide[:, :5], before[:, :5]) and torch.equal(wide[:, 5 + rows:], before[:, 5 + rows:])


@pytest.mark.parametrize("t,rows,cols,m", [("q4_k", 512, 4096, 1), ("q8_0", 256, 4096, 200), ("q5_k", 256, 4096, 30),
                                           ("q4_0", 300, 1024, 40)])
def test_residual_in_place_and_gate_in_place(t, rows, cols, m):
    wt = Weight(TYPES[t], rows, cols, 8)
    xb = syn.activation_bf16(m, cols, seed=4)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    _, mu, re = operands(m, rows, _native.F32, 10, False, True, True)
    y = re.clone()
    call(wt, x, m, y, _native.F32, 0, None, mu, y, wt.workspace(m))
    check(y, expected(wt, xb, 0, None, mu, re, _native.F32), "y is the residual")
    y = mu.clone()
    call(wt, x, m, y, _native.F32, ops.ACT_GELU, None, y, re, wt.workspace(m))
    check(y, expected(wt, xb, ops.ACT_GELU, None, mu, re, _native.F32), "y is mul")


def test_without_epilogue_the_bits_are_the_gemms():
    for t, rows, cols, m in (("q4_k", 512, 1024, 1), ("q8_0", 512, 1024, 16), ("q6_k", 14336, 512, 128),
                             ("q4_0", 300, 2048, 3), ("q8_0", 100, 2080, 40)):
        wt = Weight(TYPES[t], rows, cols, 11)
        x = torch.from_numpy(syn.activation_bf16(m, cols, seed=5).view(np.int16)).cuda()
        y = torch.empty((m, rows), device="cuda")
        ref = torch.empty((m, rows), device="cuda")
        call(wt, x, m, y, _native.F32)
        wt.handle.gemm_bf16(x.data_ptr(), m, ref.data_ptr(), stream())
        if wt.handle.linear_workspace_bytes(m) == 0:
            assert torch.equal(y.view(torch.int32), ref.view(torch.int32)), (t, rows, cols, m)


@pytest.mark.parametrize("t,rows,cols,m", [("q8_0", 256, 1024, 3), ("q4_0", 64, 512, 9), ("q4_k", 64, 512, 18),
                                           ("q5_k", 48, 512, 5), ("q6_k", 48, 512, 20), ("q6_k", 48, 512, 70)])
def test_x_off_its_usual_alignment(t, rows, cols, m):
    wt = Weight(TYPES[t], rows, cols, 12)
    xb = syn.activation_bf16(m, cols, seed=6)
    for shift in (1, 2):  # x 2 and 4 bytes past a 16-byte line
        buf = torch.zeros(m * cols + 8, device="cuda", dtype=torch.int16)
        buf[shift:shift + m * cols] = torch.from_numpy(xb.view(np.int16)).cuda().reshape(-1)
        b, mu, re = operands(m, rows, _native.BF16, 2, True, True, True)
        y = torch.empty((m, rows), device="cuda", dtype=torch.bfloat16)
        call(wt, buf[shift:], m, y, _native.BF16, ops.ACT_SILU, b, mu, re, wt.workspace(m))
        check(y, expected(wt, xb, ops.ACT_SILU, b, mu, re, _native.BF16), f"x + {2 * shift} bytes")


def test_workspaces_of_every_size_split_less():
    rows, cols, m = 256, 4096, 40
    wt = Weight(syn.Q4_K, rows, cols, 13)
    xb = syn.activation_bf16(m, cols, seed=7)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    exp = expected(wt, xb, 0, None, None, None, _native.F32)
    need = wt.handle.linear_workspace_bytes(m)
    assert need >= 2 * m * rows * 4  # this shape splits
    for size in (0, 256, m * rows * 4, 2 * m * rows * 4, need):
        ws = torch.full((max(size, 256),), 255, device="cuda", dtype=torch.uint8)  # NaNs, if they were read
        y = torch.empty((m, rows), device="cuda")
        wt.handle.linear(x.data_ptr(), m, y.data_ptr(), _native.F32, ws_ptr=ws.data_ptr(), ws_bytes=size, stream=stream())
        check(y, exp, f"workspace of {size} bytes")


def test_infinities_and_nans_of_the_operands():
    rows, cols, m = 64, 256, 6
    wt = Weight(syn.Q8_0, rows, cols, 14)
    xb = syn.activation_bf16(m, cols, seed=8)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    b, mu, re = operands(m, rows, _native.F32, 3, True, True, True)
    b[0], b[1], b[2], re[:, 3], mu[:, 4] = float("inf"), -float("inf"), float("nan"), float("inf"), float("nan")
    y = torch.empty((m, rows), device="cuda")
    call(wt, x, m, y, _native.F32, ops.ACT_RELU, b, torch.abs(mu), re, None)
    got = y.cpu().numpy()
    assert (got[:, 0] == np.inf).all()
    assert np.array_equal(got[:, 1], re[:, 1].cpu().numpy())  # relu(-inf) * |mul| + residual
    assert np.isnan(got[:, 2]).all() and (got[:, 3] == np.inf).all() and np.isnan(got[:, 4]).all()
    assert np.isfinite(got[:, 5:]).all()
    # far below zero the smooth activations end at -0 or 0, not NaN
    b.fill_(-1000.0)
    for act in (ops.ACT_SILU, ops.ACT_GELU, ops.ACT_GELU_TANH):
        call(wt, x, m, y, _native.F32, act, b)
        assert (y == 0).all()


def test_compacted_and_prepared_weights():
    rows, cols = 1024, 1024
    wt = Weight(syn.Q4_K, rows, cols, 15)
    t = ops.GgufTensor("w", (cols, rows), syn.Q4_K, wt.data.reshape(-1))
    xb = syn.activation_bf16(3, cols, seed=9)
    y0 = ops.linear(t, xb, _native.F32, activation=ops.ACT_SILU)
    t.prepare()
    y1 = ops.linear(t, xb, _native.F32, activation=ops.ACT_SILU)
    t.compact()
    y2 = ops.linear(t, xb, _native.F32, activation=ops.ACT_SILU)
    assert np.array_equal(y0, y1) and np.array_equal(y0, y2)
    # (a relative bound would not do: far below zero silu(v) turns an error of e
    # in v into one of e of its value, whatever v's own size)
    check(torch.from_numpy(y2), expected(wt, xb, ops.ACT_SILU, None, None, None, _native.F32), "compacted")
    with pytest.raises(ops.UnsupportedOperationError):
        ops.linear(t, syn.activation_bf16(9, cols, seed=1))
    t.close()


@pytest.mark.parametrize("y_type,dtype", [(_native.F32, np.float32), (_native.F16, np.float16), (_native.BF16, np.uint16)])
def test_host_form(y_type, dtype):
    rows, cols, m = 100, 512, 12
    wt = Weight(syn.Q5_K, rows, cols, 16)
    t = ops.GgufTensor("w", (cols, rows), syn.Q5_K, wt.data.reshape(-1))
    xb = syn.activation_bf16(m, cols, seed=10)
    b, mu, re = operands(m, rows, y_type, 4, True, True, True)

    def host(v):
        v = v.cpu()
        return v.view(torch.int16).numpy().view(np.uint16) if v.dtype == torch.bfloat16 else v.numpy()

    y = ops.linear(t, xb, y_type, bias=host(b), activation=ops.ACT_GELU, mul=host(mu), residual=host(re))
    assert y.dtype == dtype and y.shape == (m, rows)
    got = torch.from_numpy(y.view(np.int16)).view(torch.bfloat16) if y_type == _native.BF16 else torch.from_numpy(y)
    check(got, expected(wt, xb, ops.ACT_GELU, b, mu, re, y_type), "host form")
    assert ops.linear(t, xb[:0], y_type).shape == (0, rows)
    t.close()


def test_captured_calls_replay():
    """Two graphs with a workspace each, replayed in turn with eager work between."""
    rows, cols = 256, 4096
    wt = Weight(syn.Q8_0, rows, cols, 17)
    up = Weight(syn.Q4_K, rows, cols, 18)
    graphs, pool = [], torch.cuda.Stream()
    for m in (1, 40):
        x = torch.zeros((m, cols), device="cuda", dtype=torch.bfloat16)
        u = torch.empty((m, rows), device="cuda", dtype=torch.bfloat16)
        y = torch.empty_like(u)
        ws = torch.zeros(max(wt.handle.linear_workspace_bytes(m), up.handle.linear_workspace_bytes(m), 256), device="cuda",
                         dtype=torch.uint8)

        def gated(s, x=x, u=u, y=y, ws=ws, m=m):
            call(up, x, m, u, _native.BF16, 0, None, None, None, ws, stream=s)
            call(wt, x, m, y, _native.BF16, ops.ACT_SILU, None, u, None, ws, stream=s)

        torch.cuda.synchronize()
        with torch.cuda.stream(pool):
            gated(pool.cuda_stream)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=pool):
            gated(pool.cuda_stream)
        graphs.append((g, x, y, m, gated))
    for turn in range(3):
        for g, x, y, m, gated in graphs:
            xb = syn.activation_bf16(m, cols, seed=20 + turn)
            x.copy_(torch.from_numpy(xb.view(np.int16)).cuda().view(torch.bfloat16))
            torch.cuda.synchronize()
            y.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            got = y.clone()
            gated(stream())
            torch.cuda.synchronize()
            assert torch.equal(got.view(torch.int16), y.view(torch.int16)), (turn, m)
            x64 = (xb.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
            want = activate(ops.ACT_SILU, x64 @ wt.w.T) * (x64 @ up.w.T)
            assert o.rel_err(got.float().cpu().numpy(), want) <= 2e-2  # three bf16 roundings


def test_calls_on_two_streams_at_once():
    rows, cols, m = 256, 4096, 40
    wt = Weight(syn.Q4_K, rows, cols, 19)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = []
    for i, s in enumerate(side):
        xb = syn.activation_bf16(m, cols, seed=30 + i)
        x = torch.from_numpy(xb.view(np.int16)).cuda()
        runs.append((s, x, torch.empty((m, rows), device="cuda"), wt.workspace(m), xb))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, x, y, ws, _ in runs:
            call(wt, x, m, y, _native.F32, ops.ACT_RELU, None, None, None, ws, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for _, _, y, _, xb in runs:
        check(y, expected(wt, xb, ops.ACT_RELU, None, None, None, _native.F32), "two streams")


def test_refusals():
    rows, cols, m = 64, 256, 4
    wt = Weight(syn.Q8_0, rows, cols, 21)
    x = torch.zeros((m, cols), device="cuda", dtype=torch.int16)
    y = torch.zeros((m, 2 * rows), device="cuda")
    ws = wt.workspace(m)
    xp, yp = x.data_ptr(), y.data_ptr()

    def refused(kind, *a, **k):
        with pytest.raises(kind):
            wt.handle.linear(*a, **k)

    bad = ops.IllegalArgumentError
    refused(ops.NullPointerError, 0, m, yp, _native.F32)
    refused(ops.NullPointerError, xp, m, 0, _native.F32)
    refused(ops.UnsupportedOperationError, xp, m, yp, 8)
    refused(bad, xp, -1, yp, _native.F32)
    for act in (-1, 5):
        refused(bad, xp, m, yp, _native.F32, activation=act)
    refused(bad, xp, m, yp, _native.F32, y_stride=rows - 1)
    refused(bad, xp, m, yp, _native.F32, mul_ptr=yp + 8 * rows * m, mul_stride=rows - 1)
    refused(bad, xp, m, yp, _native.F32, residual_ptr=yp, residual_stride=2 * rows)  # y, at another stride
    refused(bad, xp, m, yp + 4, _native.F32, residual_ptr=yp)                         # one element off
    refused(bad, xp, m, yp, _native.F32, mul_ptr=yp + 4 * rows // 2, y_stride=2 * rows, mul_stride=2 * rows)
    refused(bad, xp, m, yp + 2, _native.F32)
    refused(bad, xp, m, yp + 1, _native.BF16)
    refused(bad, xp, m, yp, _native.F32, residual_ptr=yp + 2)
    refused(bad, xp + 1, m, yp, _native.F32)
    refused(bad, xp, m, yp, _native.F32, bias_ptr=yp + 2)
    refused(bad, xp, m, xp, _native.BF16)  # y over x
    refused(bad, xp, m, yp, _native.F32, ws_ptr=ws.data_ptr() + 16, ws_bytes=16)
    refused(bad, xp, m, yp, _native.F32, ws_ptr=ws.data_ptr(), ws_bytes=-1)
    wt.handle.linear(xp, 0, yp, _native.F32, stream=stream())  # nothing to do
    # the two halves of one wider matrix do not overlap
    wt.handle.linear(xp, m, yp, _native.F32, mul_ptr=yp + 4 * rows, y_stride=2 * rows, mul_stride=2 * rows, stream=stream())
    torch.cuda.synchronize()
    assert wt.handle.linear_workspace_bytes(-1) == -1 and wt.handle.linear_workspace_bytes(0) == 0
    t = ops.GgufTensor("w", (cols, rows), syn.Q8_0, wt.data.reshape(-1))
    for kw in ({"bias": np.zeros(rows + 1, np.float32)}, {"mul": np.zeros((m, rows), np.float64)},
               {"residual": np.zeros((m, rows + 1), np.float32)}, {"activation": 9}):
        with pytest.raises(bad):
            ops.linear(t, np.zeros((m, cols), np.uint16), **kw)
    with pytest.raises(bad):
        ops.linear(t, np.zeros((m, cols + 1), np.uint16))
    with pytest.raises(ops.UnsupportedOperationError):
        ops.linear(t, np.zeros((m, cols), np.uint16), 7)
    lib, e = _native.load(), _native.ErrBuf()
    xs, ys = np.zeros(m * cols, np.uint16), np.zeros(m * rows, np.float32)
    args = (t.handle(), xs.ctypes.data, xs.size, m, None, 0, None, None, ys.ctypes.data, _native.F32)
    assert lib.gollek_hip_linear(*args, ys.size - 1, e.buf, e.size) == _native.ERR_ARG
    assert lib.gollek_hip_linear(*args[:2], xs.size - 1, *args[3:], ys.size, e.buf, e.size) == _native.ERR_ARG
    assert ctypes.sizeof(ctypes.c_void_p) == 8
    t.close()


@pytest.mark.parametrize("t,rows,cols,m", [("q8_0", 256, 2880, 8), ("q8_0", 130, 2912, 70), ("q4_0", 256, 2816, 40),
                                           ("q4_0", 131, 11008, 17), ("q8_0", 97, 11008, 50), ("q4_k", 256, 2816, 16),
                                           ("q5_k", 259, 3840, 33), ("q6_k", 255, 2816, 9), ("q4_k", 130, 11008, 7)])
def test_uneven_splits_of_k(t, rows, cols, m):
    """K in parts of unequal length, outputs that are no multiple of four."""
    wt = Weight(TYPES[t], rows, cols, 23)
    assert wt.handle.linear_workspace_bytes(m) >= 2 * 4 * m * rows
    xb = syn.activation_bf16(m, cols, seed=m)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    for y_type in (_native.F32, _native.F16):
        b, mu, re = operands(m, rows, y_type, 6, True, True, True)
        y = re.clone()
        call(wt, x, m, y, y_type, ops.ACT_GELU_TANH, b, mu, y, wt.workspace(m))
        check(y, expected(wt, xb, ops.ACT_GELU_TANH, b, mu, re, y_type), f"{t} {rows}x{cols} m={m} type {y_type}")


# The mat-vec's 16-row tiles at one token: Q6_K with one and with several
# superblocks a wave, rows from one to several tiles a workgroup, and Q4_K
# beyond 64 rows a compute unit; in place, unaligned y, no workspace.
@pytest.mark.parametrize("t,rows,cols", [("q6_k", 1, 2048), ("q6_k", 17, 4096), ("q6_k", 500, 2048), ("q6_k", 4100, 4096),
                                         ("q6_k", 16, 6144), ("q6_k", 333, 14336), ("q6_k", 9000, 2048),
                                         ("q4_k", 16400, 256), ("q4_k", 20001, 512), ("q4_k", 16390, 4096)])
@pytest.mark.parametrize("y_type", [_native.F32, _native.BF16])
def test_one_token_on_row_tiles(t, rows, cols, y_type):
    print(f"[gpu] linear {t} {rows}x{cols} m=1 type={y_type}", flush=True)
    wt = Weight(TYPES[t], rows, cols, 17)
    xb = syn.activation_bf16(1, cols, seed=rows)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    b, mu, re = operands(1, rows, y_type, cols, True, True, True)
    out = torch.full((rows + 2,), 7.0, device="cuda", dtype=DTYPE[y_type])
    y = out[1:rows + 1]
    y.copy_(re[0])
    call(wt, x, 1, y, y_type, ops.ACT_SILU, b, mu, y)
    check(y.reshape(1, rows), expected(wt, xb, ops.ACT_SILU, b, mu, re, y_type), f"{t} {rows}x{cols}")
    assert out[0] == 7.0 and out[-1] == 7.0
    call(wt, x, 1, y, y_type)
    check(y.reshape(1, rows), expected(wt, xb, 0, None, None, None, y_type), f"{t} {rows}x{cols} alone")
    if y_type == _native.F32:  # the mat-vec's own sums, bit for bit
        xf = torch.from_numpy((xb.astype(np.uint32) << 16).view(np.float32)).cuda()
        ref = torch.empty(rows, device="cuda")
        wt.handle.matvec(xf.data_ptr(), ref.data_ptr(), stream=stream())
        assert torch.equal(y.view(torch.int32), ref.view(torch.int32))
    xb[0, cols // 2] = 0x7FC0  # a NaN in x reaches every sum
    call(wt, torch.from_numpy(xb.view(np.int16)).cuda(), 1, y, y_type)
    assert torch.isnan(y).all() and out[0] == 7.0 and out[-1] == 7.0


def test_more_rows_than_a_grid_axis():
    # a tall and narrow product that splits K: more than 65535 rows go through the reduction
    rows, cols, m = 8, 4096, 66560
    print(f"[gpu] linear q8_0 {rows}x{cols} m={m}", flush=True)
    wt = Weight(syn.Q8_0, rows, cols, 18)
    assert wt.handle.linear_workspace_bytes(m) >= 2 * m * rows * 4
    some = syn.activation_bf16(64, cols, seed=18)
    x = torch.from_numpy(some.view(np.int16)).cuda().repeat(m // 64, 1)
    re = torch.from_numpy(np.random.default_rng(18).normal(size=(64, rows)).astype(np.float32)).to(torch.bfloat16).cuda()
    y = re.repeat(m // 64, 1)
    call(wt, x, m, y, _native.BF16, ops.ACT_SILU, None, None, y, wt.workspace(m))
    want, tol = expected(wt, some, ops.ACT_SILU, None, None, re, _native.BF16)
    check(y, (np.tile(want, (m // 64, 1)), np.tile(tol, (m // 64, 1))), "tall")


@pytest.mark.parametrize("t,rows,cols,m", [("q4_k", 300, 512, 3), ("q8_0", 256, 512, 20), ("q6_k", 160, 512, 70),
                                           ("q4_0", 256, 4096, 40)])
def test_16_bit_operands_in_place(t, rows, cols, m):
    wt = Weight(TYPES[t], rows, cols, 19)
    xb = syn.activation_bf16(m, cols, seed=19)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    for y_type in (_native.BF16, _native.F16):
        b, mu, re = operands(m, rows, y_type, 19, True, True, True)
        y = re.clone()
        call(wt, x, m, y, y_type, ops.ACT_SILU, b, mu, y, wt.workspace(m))
        check(y, expected(wt, xb, ops.ACT_SILU, b, mu, re, y_type), "y is the residual")
        y = mu.clone()
        call(wt, x, m, y, y_type, ops.ACT_SILU, b, y, y, wt.workspace(m))
        check(y, expected(wt, xb, ops.ACT_SILU, b, mu, mu, y_type), "y is mul and the residual")


def test_output_over_its_bias_or_workspace_is_refused():
    rows, cols, m = 64, 256, 4
    wt = Weight(syn.Q8_0, rows, cols, 22)
    x = torch.zeros((m, cols), device="cuda", dtype=torch.int16)
    y = torch.zeros(m * rows + 256, device="cuda")
    yp = (y.data_ptr() + 255) // 256 * 256
    for kw in ({"bias_ptr": yp}, {"bias_ptr": yp + 4 * (m * rows - 1)}, {"bias_ptr": yp - 4 * (rows - 1)},
               {"ws_ptr": yp, "ws_bytes": 256}, {"ws_ptr": yp - 256, "ws_bytes": 512}):
        with pytest.raises(ops.IllegalArgumentError):
            wt.handle.linear(x.data_ptr(), m, yp, _native.F32, **kw)
    room = torch.zeros(512 + m * rows + rows, device="cuda")
    zp = (room.data_ptr() + 255) // 256 * 256 + 4 * rows
    for bias in (zp - 4 * rows, zp + 4 * m * rows):  # right before it, right behind it
        wt.handle.linear(x.data_ptr(), m, zp, _native.F32, bias_ptr=bias, ws_ptr=zp - 4 * rows, ws_bytes=4 * rows,
                         stream=stream())
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows,cols", [(64, 8192), (1000, 8192), (320, 14336)])
def test_one_token_of_few_long_rows_with_and_without_a_workspace(rows, cols):
    wt = Weight(syn.Q6_K, rows, cols, 23)
    xb = syn.activation_bf16(1, cols, seed=23)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    b, mu, re = operands(1, rows, _native.BF16, 23, True, True, True)
    want = expected(wt, xb, ops.ACT_SILU, b, mu, re, _native.BF16)
    for ws in (wt.workspace(1), None):
        y = torch.full((1, rows), float("nan"), device="cuda", dtype=torch.bfloat16)
        call(wt, x, 1, y, _native.BF16, ops.ACT_SILU, b, mu, re, ws)
        check(y, want, f"{rows}x{cols} workspace {ws is not None}")


# v Phi(v) = v erfc(z) / 2 at z = -v / sqrt(2): z by one rounded constant and one
# product, 2^-23 relative, of which erfc makes at most (2 z^2 + 2 z) 2^-23 for z > 0
# (|erfc'(z)| <= (2 z + 2 / z) erfc(z) from z = 1 on) and 2^-23 below; erfc itself
# 16 units of 2^-23 (the bound OpenCL sets its own), two products and the cast's half step.
@pytest.mark.parametrize("y_type", [_native.F32, _native.F16, _native.BF16])
@pytest.mark.parametrize("t,cols,m", [("q4_k", 512, 1), ("q8_0", 512, 20), ("q4_k", 4096, 40), ("q8_0", 32, 3),
                                      ("q8_0", 512, 100)])
def test_gelu_keeps_its_precision_below_zero(t, cols, m, y_type):
    from scipy.special import erfc

    v = np.concatenate([np.linspace(-12.5, 9.0, 498), [-0.0, 0.0, 1e-20, -1e-20, 1e30, -1e30]]).astype(np.float32)
    wt = Weight(TYPES[t], v.size, cols, 24)
    x = torch.zeros((m, cols), device="cuda", dtype=torch.int16)  # the product is 0: v is the bias alone
    for odd in (0, 1):  # whole vectors of a row, and single elements
        room = torch.full((m, v.size + 16), 7.0, device="cuda", dtype=DTYPE[y_type])
        y = room[:, odd:odd + v.size]
        call(wt, x, m, y, y_type, ops.ACT_GELU, torch.from_numpy(v).cuda(), ws=wt.workspace(m), y_stride=room.shape[1])
        v64 = v.astype(np.float64)
        want = np.where(v64 < -1e3, -0.0, 0.5 * v64 * erfc(-v64 / np.sqrt(2.0)))
        z = np.clip(-v64 / np.sqrt(2.0), 0.0, 10.0)
        rel = (2 * z * z + 2 * z + 1 + 16 + 1) * 2.0**-23 + HALF_STEP[y_type]
        over = np.abs(want) > 65504.0 if y_type == _native.F16 else np.zeros(v.size, bool)
        got = f64(y)
        assert np.isinf(got[:, over]).all() and np.isfinite(got[:, ~over]).all()
        err = np.abs(got - want)[:, ~over] - (2.0**-25 if y_type == _native.F16 else 2.0**-149)
        worst = (err / np.maximum(rel * np.abs(want), 1e-300)[~over]).max()
        print(f"[gpu] gelu {t} m={m} type={y_type}: largest error {worst:.3f} of its bound", flush=True)
        assert worst <= 1.0
        assert (room[:, odd + v.size:] == 7.0).all()


@pytest.mark.parametrize("t,rows,cols,m", [("q8_0", 1024, 14336, 1111), ("q4_0", 2048, 11008, 1129), ("q8_0", 257, 2080, 900),
                                           ("q4_k", 1024, 8192, 300), ("q6_k", 512, 8192, 1), ("q8_0", 256, 4096, 8)])
def test_a_larger_workspace_changes_no_bit(t, rows, cols, m):
    """The plan is the stated workspace's, whatever a caller has beyond it; and what is beyond stays as it is."""
    print(f"[gpu] linear {t} {rows}x{cols} m={m} larger workspace", flush=True)
    wt = Weight(TYPES[t], rows, cols, 25)
    xb = syn.activation_bf16(m, cols, seed=25)
    x = torch.from_numpy(xb.view(np.int16)).cuda()
    need = wt.handle.linear_workspace_bytes(m)
    y, z = (torch.full((m, rows), float("nan"), device="cuda") for _ in range(2))
    call(wt, x, m, y, _native.F32, ops.ACT_SILU, ws=wt.workspace(m))
    big = torch.full((need + (128 << 20),), 171, device="cuda", dtype=torch.uint8)
    call(wt, x, m, z, _native.F32, ops.ACT_SILU, ws=big)
    assert torch.equal(y.view(torch.int32), z.view(torch.int32))
    assert (big[need:] == 171).all()
    some = np.unique(np.r_[0:min(m, 20), m // 2, m - 1])
    check(z[some], expected(wt, xb[some], ops.ACT_SILU, None, None, None, _native.F32), f"{t} {rows}x{cols} m={m}")


# One to four tokens on the mat-vec's kernels and up to 32 on the skinny one never split,
# others of the same weights do: K-quants from few rows on, and a Q6_K weight of few long rows.
@pytest.mark.parametrize("t,rows,cols,never,splits", [
    ("q4_0", 300, 2048, (1, 2, 3, 4), (5, 40)), ("q4_k", 512, 8192, (1, 2), (3, 16)), ("q5_k", 256, 4096, (1, 4), (5,)),
    ("q8_0", 512, 8192, (1, 2, 3, 32), (33,)), ("q8_0", 500, 8192, (1, 2), (3, 32)), ("q6_k", 2048, 4096, (1,), (8,)),
    ("q6_k", 1024, 6144, (1,), (2,)), ("q6_k", 1024, 8192, (), (1, 2)), ("q4_k", 16400, 256, (1,), ())])
def test_no_workspace_is_asked_for_where_none_is_used(t, rows, cols, never, splits):
    wt = Weight(TYPES[t], rows, cols, 26)
    for m in never:
        assert wt.handle.linear_workspace_bytes(m) == 0, m
        x = torch.from_numpy(syn.activation_bf16(m, cols, seed=26).view(np.int16)).cuda()
        ws = torch.full((16 << 20,), 171, device="cuda", dtype=torch.uint8)
        y, z = (torch.full((m, rows), float("nan"), device="cuda") for _ in range(2))
        call(wt, x, m, y, _native.F32)
        call(wt, x, m, z, _native.F32, ws=ws)
        assert torch.equal(y.view(torch.int32), z.view(torch.int32)) and (ws == 171).all(), m
    for m in splits:
        assert wt.handle.linear_workspace_bytes(m) >= 2 * 4 * m * rows, m


def test_without_a_workspace_the_bits_are_the_gemms():
    """Shapes that the plain GEMM does not split, whatever a workspace would change."""
    for t, rows, cols, m in (("q4_0", 300, 2048, 3), ("q8_0", 100, 2080, 40), ("q4_0", 131, 2848, 300), ("q4_k", 512, 1024, 2),
                             ("q6_k", 14336, 512, 128), ("q8_0", 512, 1024, 16)):
        wt = Weight(TYPES[t], rows, cols, 27)
        x = torch.from_numpy(syn.activation_bf16(m, cols, seed=27).view(np.int16)).cuda()
        y, ref = (torch.full((m, rows), float("nan"), device="cuda") for _ in range(2))
        call(wt, x, m, y, _native.F32)
        wt.handle.gemm_bf16(x.data_ptr(), m, ref.data_ptr(), stream())
        assert torch.equal(y.view(torch.int32), ref.view(torch.int32)), (t, rows, cols, m)


@pytest.mark.parametrize("t,m", [("q4_k", 40), ("q8_0", 64)])
def test_a_workspace_over_an_input_is_refused(t, m):
    rows, cols = 256, 4096
    wt = Weight(TYPES[t], rows, cols, 28)
    need = wt.handle.linear_workspace_bytes(m)
    assert need > 0
    xb = syn.activation_bf16(m, cols, seed=28)
    b, mu, re = operands(m, rows, _native.F32, 28, True, True, True)
    size = 2 * m * cols
    room = torch.zeros(need + 4 * size, device="cuda", dtype=torch.uint8)
    base = (room.data_ptr() + 255) // 256 * 256
    y = torch.full((m, rows), 7.0, device="cuda")
    xp = torch.from_numpy(xb.view(np.int16)).cuda()
    put = dict(bias_ptr=b.data_ptr(), mul_ptr=mu.data_ptr(), residual_ptr=re.data_ptr(), stream=stream())
    for at in (base, base + need - 16):  # at the workspace's start and over its last bytes
        with pytest.raises(ops.IllegalArgumentError):
            wt.handle.linear(at, m, y.data_ptr(), _native.F32, ws_ptr=base, ws_bytes=need, **put)
        for name in ("bias_ptr", "mul_ptr", "residual_ptr"):
            with pytest.raises(ops.IllegalArgumentError):
                wt.handle.linear(xp.data_ptr(), m, y.data_ptr(), _native.F32, ws_ptr=base, ws_bytes=need, **{**put, name: at})
    torch.cuda.synchronize()
    assert (y == 7.0).all()
    # right behind what the call uses an input may stand, whatever the workspace's length
    at = base - room.data_ptr() + need
    room[at:at + size].view(torch.int16).copy_(xp.reshape(-1))
    wt.handle.linear(base + need, m, y.data_ptr(), _native.F32, ws_ptr=base, ws_bytes=need + size, activation=ops.ACT_SILU, **put)
    check(y, expected(wt, xb, ops.ACT_SILU, b, mu, re, _native.F32), "x behind the workspace")


def test_the_host_form_keeps_its_handles_small():
    """A handle's staging stays: x, y and no more than 16 MiB of partials beyond the first."""
    rows, cols, m = 2048, 11008, 1129
    wt = Weight(syn.Q4_0, rows, cols, 29)
    y_bytes = 4 * m * rows
    assert wt.handle.linear_workspace_bytes(m) > (16 << 20) + 2 * y_bytes  # the device form splits further
    t = ops.GgufTensor("w", (cols, rows), syn.Q4_0, wt.data.reshape(-1))
    xb = syn.activation_bf16(m, cols, seed=29)
    ops.linear(t, xb[:1])
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    y = ops.linear(t, xb, _native.F32, activation=ops.ACT_RELU)
    held = before - torch.cuda.mem_get_info()[0]
    assert held <= 2 * m * cols + 2 * y_bytes + (16 << 20) + (8 << 20)  # (and the allocator's granularity)
    some = np.r_[0:20, m - 1]
    check(torch.from_numpy(y[some]), expected(wt, xb[some], ops.ACT_RELU, None, None, None, _native.F32), "host form")
    t.close()
