"""Expert routing with a bias and groups against float64.

Both sides choose by scores in double, whose errors (1e-16) leave the order of
random scores alone; equal scores are planted where ties matter.  A weight is a
quotient in double (relative error below 2^-48) rounded once to fp32: half a
step, 2^-24, relative.
"""
import numpy as np
import pytest
import torch

from gollek_amd import _native
from gollek_amd import synthetic as syn
from gollek_amd import tensor_ops as ops
from oracle import oracle as o

pytestmark = pytest.mark.gpu
DTYPE = {_native.F32: torch.float32, _native.F16: torch.float16, _native.BF16: torch.bfloat16}
TOL = 2.0**-24 * (1 + 2.0**-20)


@pytest.fixture(scope="module", autouse=True)
def _init():
    ops.init(0)


def reference(logits, top_k, scoring, bias=None, n_groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0):
    """ids, weights in float64, token by token, from the definition."""
    out_i, out_w = [], []
    for l in np.asarray(logits, np.float64):
        with np.errstate(over="ignore", invalid="ignore"):
            if scoring == ops.ROUTER_SOFTMAX:
                p = np.exp(l - np.nanmax(l))
                p = p / p.sum()
            else:
                p = 1.0 / (1.0 + np.exp(-l))
        c = p if bias is None else p + np.asarray(bias, np.float64)
        n = len(l)
        above = lambda v: np.where(np.isnan(v), np.inf, v)  # noqa: E731
        nan_first = lambda i: (0 if np.isnan(c[i]) else 1, -above(c)[i], i)  # noqa: E731
        size = n // n_groups
        worth = []
        for g in range(n_groups):
            best = sorted(range(g * size, (g + 1) * size), key=nan_first)[:group_top]
            worth.append(sum(c[i] for i in best))
        groups = sorted(range(n_groups), key=lambda g: (0 if np.isnan(worth[g]) else 1, -above(np.array(worth))[g], g))
        kept = set(groups[:top_groups])
        ids = sorted((i for i in range(n) if i // size in kept), key=nan_first)[:top_k]
        w = p[ids]
        s = 0.0
        for v in w:
            s += v
        if renormalize and s > 0:
            w = w / s
        out_i.append(ids)
        out_w.append(w * scale)
    return np.array(out_i, np.int32).reshape(-1, top_k), np.array(out_w).reshape(-1, top_k)


def route(logits, top_k, scoring, bias=None, **kw):
    """The device entry on a CUDA tensor of logits."""
    n, e = logits.shape
    kind = {v: k for k, v in DTYPE.items()}[logits.dtype]
    ids = torch.full((n, top_k), -7, device="cuda", dtype=torch.int32)
    w = torch.full((n, top_k), float("nan"), device="cuda")
    b = None if bias is None else torch.as_tensor(np.asarray(bias, np.float32)).cuda()
    ops.moe_route_device(logits.data_ptr(), kind, n, e, top_k, scoring, ids.data_ptr(), w.data_ptr(),
                         bias_ptr=0 if b is None else b.data_ptr(), stream=torch.cuda.current_stream().cuda_stream, **kw)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), w.cpu().numpy()


def compare(got, want, what):
    ids, w = got
    wi, ww = want
    assert np.array_equal(ids, wi), what
    assert np.array_equal(np.isnan(w), np.isnan(ww)), what
    ok = ~np.isnan(ww)
    # (weights below fp32's normal range round to steps of 2^-149)
    assert (np.abs(w[ok] - ww[ok]) <= TOL * np.abs(ww[ok]) + 2.0**-150).all(), what


CASES = [  # tokens, experts, top_k, groups, top_groups, group_top
    (1, 8, 2, 1, 1, 1), (3, 1, 1, 1, 1, 1), (5, 60, 4, 1, 1, 1), (37, 64, 6, 1, 1, 1), (1, 128, 8, 1, 1, 1),
    (300, 128, 8, 1, 1, 1), (33, 160, 6, 8, 3, 1), (7, 256, 8, 8, 4, 2), (129, 256, 8, 8, 1, 2), (2, 384, 9, 1, 1, 1),
    (9, 96, 5, 3, 2, 2), (4, 512, 10, 16, 5, 1), (3, 1000, 12, 5, 2, 2), (2, 4096, 64, 64, 32, 2), (2, 4096, 100, 1, 1, 1),
    (3, 80, 80, 1, 1, 1), (2, 64, 7, 64, 9, 2), (5, 66, 3, 33, 2, 2), (2, 1025, 5, 1, 1, 1), (1, 513, 3, 27, 2, 1),
]


@pytest.mark.parametrize("scoring", [ops.ROUTER_SOFTMAX, ops.ROUTER_SIGMOID])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_route_matches_float64(i, scoring):
    n, e, k, g, tg, gt = CASES[i]
    print(f"[gpu] route {CASES[i]} scoring={scoring}", flush=True)
    rng = np.random.default_rng(i)
    kind = (_native.F32, _native.BF16, _native.F16)[(i + scoring) % 3]
    logits = torch.from_numpy(rng.normal(size=(n, e)).astype(np.float32) * 2).to(DTYPE[kind]).cuda()
    bias = (rng.normal(size=e) * 0.05).astype(np.float32) if i % 2 else None
    kw = dict(n_groups=g, top_groups=tg, group_top=gt, renormalize=i % 3 != 0, scale=(1.0, 2.5)[i % 2])
    compare(route(logits, k, scoring, bias, **kw),
            reference(logits.double().cpu().numpy(), k, scoring, bias, **kw), CASES[i])


def test_plain_routing_equals_select_topk():
    rng = np.random.default_rng(5)
    logits = rng.normal(size=(200, 128)).astype(np.float32)
    for scoring in (ops.ROUTER_SOFTMAX, ops.ROUTER_SIGMOID):
        ids, w = ops.moe_select_topk(logits, 8, scoring)
        ids2, w2 = ops.moe_route(logits, 8, scoring)
        assert np.array_equal(ids, ids2)
        # select_topk rounds every step to fp32: the score (sigmoid 4 steps; softmax 2,
        # and 128 in its sum), the sum of 8 and the quotient
        assert np.abs(w / w2 - 1).max() <= (2 + 128 + 4 + 8 + 1) * 2.0**-24


def test_equal_scores_go_to_the_lower_index():
    e = 256
    logits = torch.zeros((2, e), device="cuda")
    logits[1, 5::7] = 1.0
    ids, w = route(logits, 8, ops.ROUTER_SOFTMAX)
    assert ids[0].tolist() == list(range(8)) and ids[1].tolist() == [5 + 7 * j for j in range(8)]
    assert np.all(w == 0.125)
    # equal groups too: the first two
    ids, _ = route(logits[:1], 8, ops.ROUTER_SIGMOID, n_groups=8, top_groups=2, group_top=2)
    assert ids[0].tolist() == list(range(8))
    # scores that are equal in fp32 only are not ties: sigmoid(20) and sigmoid(21)
    logits = torch.full((1, 64), -5.0, device="cuda")
    logits[0, 3], logits[0, 9] = 20.0, 21.0
    ids, _ = route(logits, 2, ops.ROUTER_SIGMOID)
    assert ids[0].tolist() == [9, 3]
    # both round to 1 in double: a tie
    logits[0, 3], logits[0, 9] = 40.0, 41.0
    ids, _ = route(logits, 2, ops.ROUTER_SIGMOID)
    assert ids[0].tolist() == [3, 9]


@pytest.mark.parametrize("scoring", [ops.ROUTER_SOFTMAX, ops.ROUTER_SIGMOID])
def test_masked_infinite_and_nan_logits(scoring):
    inf, nan = float("inf"), float("nan")
    rng = np.random.default_rng(6)
    l = rng.normal(size=(7, 64)).astype(np.float32)
    l[0, :60] = -inf           # four experts left
    l[1, 1:] = -inf            # one left: the others' weight is 0
    l[2, 17] = nan
    l[3, [3, 40]] = inf
    l[4] = -3.0e38
    l[5] = -inf                # nothing left: softmax NaN, sigmoid 0
    l[6, 2] = 3.0e38
    kw = dict(n_groups=4, top_groups=3, group_top=2)
    with np.errstate(all="ignore"):
        # (np.nanmax of an all -inf row is -inf: NaN scores, as the definition has it)
        compare(route(torch.from_numpy(l).cuda(), 6, scoring), reference(l, 6, scoring), "no groups")
        compare(route(torch.from_numpy(l).cuda(), 6, scoring, **kw), reference(l, 6, scoring, **kw), "groups")
    bias = np.zeros(64, np.float32)
    bias[:62] = -inf           # a bias can rule experts out; the order of those is by index
    compare(route(torch.from_numpy(l[:1]).cuda(), 4, scoring, bias), reference(l[:1], 4, scoring, bias), "bias -inf")


def test_weights_of_zero_sum_are_not_divided():
    l = torch.full((1, 16), -float("inf"), device="cuda")
    _, w = route(l, 4, ops.ROUTER_SIGMOID, renormalize=True, scale=3.0)
    assert (w == 0).all()


def test_captured_route_replays():
    n, e, k = 50, 128, 8
    logits = torch.zeros((n, e), device="cuda")
    ids = torch.zeros((n, k), device="cuda", dtype=torch.int32)
    w = torch.zeros((n, k), device="cuda")
    s = torch.cuda.Stream()

    def go(st):
        ops.moe_route_device(logits.data_ptr(), _native.F32, n, e, k, 0, ids.data_ptr(), w.data_ptr(), n_groups=8,
                             top_groups=4, stream=st)

    with torch.cuda.stream(s):
        go(s.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        go(s.cuda_stream)
    for turn in range(3):
        l = np.random.default_rng(turn).normal(size=(n, e)).astype(np.float32)
        logits.copy_(torch.from_numpy(l).cuda())
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        compare((ids.cpu().numpy(), w.cpu().numpy()), reference(l, k, 0, n_groups=8, top_groups=4), turn)


@pytest.mark.parametrize("tokens", [1, 9, 100])
def test_routed_block_is_the_route_and_the_experts(tokens):
    e, h, inter, k = 16, 256, 256, 4
    rng = np.random.default_rng(tokens)
    dev = {}
    for name, rows, cols in (("gate", e * inter, h), ("up", e * inter, h), ("down", e * h, inter)):
        d = syn.matrix(syn.Q4_K, rows, cols, seed=len(name))
        t = torch.from_numpy(d.reshape(-1)).cuda()
        dev[name] = (t, ops.DeviceWeight(syn.Q4_K, t.data_ptr(), rows, cols), d)
    x = torch.from_numpy(rng.normal(size=(tokens, h)).astype(np.float32)).cuda()
    logits = torch.from_numpy(rng.normal(size=(tokens, e)).astype(np.float32)).to(torch.bfloat16).cuda()
    bias = torch.from_numpy((0.1 * rng.normal(size=e)).astype(np.float32)).cuda()
    kw = dict(n_groups=4, top_groups=2, group_top=2, scale=1.5)
    ids = torch.zeros((tokens, k), device="cuda", dtype=torch.int32)
    w, out, out2 = (torch.zeros(s, device="cuda") for s in ((tokens, k), (tokens, h), (tokens, h)))
    ws = torch.zeros(ops.moe_workspace_bytes(tokens, k, h, inter, e), device="cuda", dtype=torch.uint8)
    st = torch.cuda.current_stream().cuda_stream
    gw, uw, dw = (dev[n][1] for n in ("gate", "up", "down"))
    ops.moe_block_routed_device(gw, uw, dw, e, x.data_ptr(), logits.data_ptr(), _native.BF16, tokens, k,
                                ops.ROUTER_SIGMOID, ids.data_ptr(), w.data_ptr(), out.data_ptr(), ws.data_ptr(),
                                ws.numel(), bias_ptr=bias.data_ptr(), stream=st, **kw)
    want = reference(logits.double().cpu().numpy(), k, ops.ROUTER_SIGMOID, bias.cpu().numpy(), **kw)
    compare((ids.cpu().numpy(), w.cpu().numpy()), want, "block's routes")
    ops.moe_grouped_device(gw, uw, dw, e, x.data_ptr(), ids.data_ptr(), w.data_ptr(), tokens, k, out2.data_ptr(),
                           ws.data_ptr(), ws.numel(), st)
    torch.cuda.synchronize()
    assert torch.equal(out, out2)
    m = {n: o.dequantize(syn.Q4_K, dev[n][2], c).astype(np.float64).reshape(e, r, c)
         for n, r, c in (("gate", inter, h), ("up", inter, h), ("down", h, inter))}
    xs = x.double().cpu().numpy()
    ref = np.zeros((tokens, h))
    for t in range(tokens):
        for i, wt in zip(*(a[t] for a in want)):
            a = m["gate"][i] @ xs[t]
            ref[t] += wt * (m["down"][i] @ (a / (1 + np.exp(-np.clip(a, -700, 700))) * (m["up"][i] @ xs[t])))
    assert o.rel_err(out.cpu().numpy().reshape(-1), ref.reshape(-1)) <= 1e-3  # the expert passes' parity bar


def test_host_form_and_refusals():
    rng = np.random.default_rng(8)
    l = rng.normal(size=(6, 32)).astype(np.float32)
    b = (0.1 * rng.normal(size=32)).astype(np.float32)
    kw = dict(n_groups=4, top_groups=2, group_top=2, scale=0.5)
    compare(ops.moe_route(l, 4, 1, bias=b, **kw), reference(l, 4, 1, b, **kw), "host")
    h = l.astype(np.float16)
    compare(ops.moe_route(h, 4, 0), reference(h, 4, 0), "host fp16")
    ids, w = ops.moe_route(l[:0], 4, 0)
    assert ids.shape == w.shape == (0, 4)
