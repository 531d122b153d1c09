"""Sampling against its definition in float64, row by row.

Tokens and kept counts are compared exactly: the kernel sums weights as
multiples of 2^-S (V 2^S < 2^62), so its masses are off by at most V 2^-(S + 1)
of the largest weight (4e-9 at 128k), and the settings and random numbers of
these cases lie further than that from a border.  A probability is
a quotient of a weight in double and such a mass, rounded once to fp32: 2^-24
and V 2^-(S + 1) relative.
"""
import numpy as np
import pytest
import torch

from gollek_amd import _native
from gollek_amd import synthetic as syn
from gollek_amd import tensor_ops as ops

pytestmark = pytest.mark.gpu
DTYPE = {_native.F32: torch.float32, _native.F16: torch.float16, _native.BF16: torch.bfloat16}
KIND = {v: k for k, v in DTYPE.items()}


@pytest.fixture(scope="module", autouse=True)
def _init():
    ops.init(0)


def reference(l, u, t=1.0, k=0, p=1.0, mp=0.0):
    """token, prob, kept of one row of float64 logits."""
    at = np.flatnonzero(l > -np.inf)  # (NaN compares false)
    if not at.size:
        return -1, 0.0, 0
    at = at[np.lexsort((at, -l[at]))]
    if not t > 0:
        at, t = at[:1], 1.0
    if k > 0:
        at = at[:k]
    if np.isinf(l[at[0]]):
        w = (l[at] == np.inf).astype(np.float64)
    else:
        w = np.exp((l[at] - l[at[0]]) / t)
    if p < 1:
        mass = np.cumsum(w)
        n = 1 if not p > 0 else int((mass < p * mass[-1]).sum()) + 1
        at, w = at[:n], w[:n]
    if mp > 0:
        keep = w >= min(mp, 1.0)
        at, w = at[keep], w[keep]
    order = np.argsort(at)
    at, w = at[order], w[order]
    mass = np.cumsum(w)
    u = min(max(0.0 if np.isnan(u) else u, 0.0), 1 - 2.0**-24)
    i = int((mass <= u * mass[-1]).sum())
    return int(at[i]), w[i] / mass[-1], at.size


def sample(logits, u, t=None, k=None, p=None, mp=None, vocab=None, stream=None):
    """The device entry on a CUDA tensor of logits (rows may be longer than vocab)."""
    rows, stride = logits.shape
    vocab = stride if vocab is None else vocab

    def dev(v, dtype):
        return None if v is None else torch.as_tensor(np.broadcast_to(np.asarray(v, dtype), (rows,)).copy()).cuda()

    t, k, p, mp, u = dev(t, np.float32), dev(k, np.int32), dev(p, np.float32), dev(mp, np.float32), dev(u, np.float32)
    tok = torch.full((rows,), -9, device="cuda", dtype=torch.int32)
    kept = torch.full((rows,), -9, device="cuda", dtype=torch.int32)
    prob = torch.full((rows,), float("nan"), device="cuda")
    ws = torch.full((max(ops.sample_workspace_bytes(rows, vocab), 256),), 255, device="cuda", dtype=torch.uint8)
    at = [0 if v is None else v.data_ptr() for v in (t, k, p, mp)]
    ops.sample_device(logits.data_ptr(), KIND[logits.dtype], rows, vocab, u.data_ptr(), tok.data_ptr(),
                      logits_stride=stride, temperature_ptr=at[0], top_k_ptr=at[1], top_p_ptr=at[2], min_p_ptr=at[3],
                      probs_ptr=prob.data_ptr(), kept_ptr=kept.data_ptr(), ws_ptr=ws.data_ptr(), ws_bytes=ws.numel(),
                      stream=torch.cuda.current_stream().cuda_stream if stream is None else stream)
    torch.cuda.synchronize()
    return tok.cpu().numpy(), prob.cpu().numpy(), kept.cpu().numpy()


def compare(got, l, u, what, t=1.0, k=0, p=1.0, mp=0.0):
    l = l.double().cpu().numpy() if torch.is_tensor(l) else np.asarray(l, np.float64)
    rows, v = l.shape
    f32 = lambda x: np.broadcast_to(np.asarray(x, np.float32).astype(np.float64), (rows,))  # noqa: E731
    u, t, p, mp, k = f32(u), f32(t), f32(p), f32(mp), np.broadcast_to(np.asarray(k), (rows,))
    tol = 2.0**-24 * 1.01 + v * 2.0 ** -(62 - v.bit_length() + 1)
    for r in range(rows):
        token, prob, kept = reference(l[r], u[r], t[r], int(k[r]), p[r], mp[r])
        have = (int(got[0][r]), float(got[1][r]), int(got[2][r]))
        print(f"[gpu] {what} row {r}: {have} want {(token, prob, kept)}", flush=True)
        assert have[0] == token and have[2] == kept, (what, r)
        assert abs(have[1] - prob) <= tol * prob + 2.0**-150, (what, r)


def logits_of(rows, vocab, seed, dtype=torch.float32, sigma=2.5):
    rng = np.random.default_rng(seed)
    l = rng.normal(size=(rows, vocab)) * sigma
    for r in range(rows):
        l[r, rng.integers(0, vocab, 12)] = rng.uniform(6, 14, 12)
    return torch.from_numpy(l.astype(np.float32)).to(dtype).cuda()


SETTINGS = [dict(), dict(t=0.7), dict(t=1.4, k=40), dict(p=0.9), dict(t=0.8, k=40, p=0.95), dict(mp=0.05),
            dict(t=1.3, k=300, p=0.8, mp=0.01), dict(t=0.0), dict(k=1), dict(t=0.01, p=0.99), dict(t=30.0, p=0.5),
            dict(t=100.0, k=5000, p=0.9), dict(t=3.0, p=0.97, mp=1e-4), dict(t=50.0, mp=0.7)]


@pytest.mark.parametrize("i", range(len(SETTINGS)))
@pytest.mark.parametrize("vocab,rows", [(1, 2), (2, 5), (63, 9), (1000, 6), (1025, 4), (4097, 3), (32000, 3),
                                        (128256, 2)])
def test_sample_matches_float64(vocab, rows, i):
    dtype = (torch.float32, torch.bfloat16, torch.float16)[(i + vocab) % 3]
    l = logits_of(rows, vocab, 10 * i + vocab, dtype)
    u = np.random.default_rng(i).random(rows).astype(np.float32)
    compare(sample(l, u, **SETTINGS[i]), l, u, f"{vocab} {SETTINGS[i]} {dtype}", **SETTINGS[i])


def test_a_batch_with_settings_of_its_own_and_a_stride():
    rows, vocab, stride = 70, 5001, 5056
    wide = logits_of(rows, stride, 3)
    wide[:, vocab:] = 1e4  # behind the vocabulary: never read as a token
    rng = np.random.default_rng(4)
    kw = dict(t=rng.choice([0.0, 0.6, 1.0, 1.7], rows), k=rng.choice([0, -3, 1, 7, 50, 900, 10**6], rows),
              p=rng.choice([0.5, 0.9, 0.99, 1.0, 1.5], rows), mp=rng.choice([0.0, -1.0, 0.02, 0.3], rows))
    u = rng.random(rows).astype(np.float32)
    compare(sample(wide, u, vocab=vocab, **kw), wide[:, :vocab], u, "batch", **kw)


def test_the_random_number_runs_through_the_distribution():
    l = logits_of(1, 300, 5, sigma=1.0)
    u = np.concatenate([[0.0, 1 - 2.0**-24, 1.0, 2.0, -1.0, np.nan], np.linspace(0.001, 0.999, 500)]).astype(np.float32)
    many = l.expand(u.size, -1).contiguous()
    got = sample(many, u, k=60, p=0.9)
    compare(got, many, u, "u", k=60, p=0.9)
    kept = got[2][0]
    assert (got[2] == kept).all() and len(set(got[0].tolist())) > kept // 2


@pytest.mark.parametrize("vocab", [500, 40000])
def test_equal_logits(vocab):
    """Ties are kept by index, in every filter."""
    u = np.array([0.0, 0.3, 0.77, 0.999], np.float32)
    flat = torch.zeros((4, vocab), device="cuda")
    for kw in (dict(), dict(k=37), dict(p=0.301), dict(k=200, p=0.503), dict(mp=0.9), dict(p=0.999, t=2.0)):
        compare(sample(flat, u, **kw), flat, u, f"flat {kw}", **kw)
    steps = (torch.arange(vocab, device="cuda") * 7919 % 5).float().expand(4, -1).contiguous()  # five values
    steps[:, 1::2] *= -0.0  # and zeros of both signs
    for kw in (dict(k=vocab // 3), dict(p=0.6003), dict(k=vocab // 2 + 1, p=0.8501, t=0.9), dict(mp=0.03)):
        compare(sample(steps, u, **kw), steps, u, f"steps {kw}", **kw)


def test_masked_empty_nan_and_infinite_rows():
    inf, nan = float("inf"), float("nan")
    vocab = 2050
    l = logits_of(8, vocab, 6)
    l[0] = -inf                                # nothing left
    l[1, 1:] = -inf                            # one token
    l[2] = nan
    l[3, ::2] = nan                            # NaN is no token, wherever it stands
    l[4, 100] = l[4, 2000] = inf               # two infinite ones share the weight
    l[5, torch.arange(vocab) % 50 != 7] = -inf
    l[6] = -3.0e38
    l[7, :3] = torch.tensor([3.3e38, 3.4e38, -3.4e38])
    u = np.full(8, 0.6, np.float32)
    for kw in (dict(), dict(k=5), dict(p=0.7), dict(t=0.9, k=30, p=0.9, mp=0.02), dict(t=0.0), dict(t=nan),
               dict(t=inf, k=100, p=0.33), dict(t=1e-44), dict(p=0.0), dict(p=-1.0), dict(p=nan, mp=nan), dict(mp=5.0)):
        ref = dict(kw)
        if kw.get("p") is not None and np.isnan(kw.get("p")):
            ref.pop("p"), ref.pop("mp")  # neither is below 1 nor above 0: off
        compare(sample(l, u, **kw), l, u, f"{kw}", **ref)


def test_a_rows_token_does_not_depend_on_its_batch():
    vocab = 33000
    l = logits_of(130, vocab, 7)
    u = np.random.default_rng(8).random(130).astype(np.float32)
    for kw in (dict(t=1.1), dict(p=0.95), dict(k=80, p=0.9)):
        all_rows = sample(l, u, **kw)
        for r in (0, 64, 129):
            one = sample(l[r:r + 1].contiguous(), u[r:r + 1], **kw)
            assert [a[0] for a in one] == [a[r] for a in all_rows]
        again = sample(l, u, **kw)
        assert all(np.array_equal(a, b) for a, b in zip(all_rows, again))


def test_captured_calls_replay():
    rows, vocab = 3, 40000
    kw = dict(t=0.9, k=50, p=0.9)
    l = torch.zeros((rows, vocab), device="cuda")
    u = torch.zeros(rows, device="cuda")
    par = [torch.full((rows,), v, device="cuda", dtype=d) for v, d in ((0.9, torch.float32), (50, torch.int32),
                                                                      (0.9, torch.float32))]
    tok = torch.zeros(rows, device="cuda", dtype=torch.int32)
    kept, prob = torch.zeros_like(tok), torch.zeros(rows, device="cuda")
    ws = torch.zeros(max(ops.sample_workspace_bytes(rows, vocab), 256), device="cuda", dtype=torch.uint8)
    s = torch.cuda.Stream()

    def go(stream):
        ops.sample_device(l.data_ptr(), _native.F32, rows, vocab, u.data_ptr(), tok.data_ptr(),
                          temperature_ptr=par[0].data_ptr(), top_k_ptr=par[1].data_ptr(), top_p_ptr=par[2].data_ptr(),
                          probs_ptr=prob.data_ptr(), kept_ptr=kept.data_ptr(), ws_ptr=ws.data_ptr(),
                          ws_bytes=ws.numel(), stream=stream)

    with torch.cuda.stream(s):
        go(s.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        go(s.cuda_stream)
    for turn in range(4):
        new = logits_of(rows, vocab, 50 + turn)
        nu = np.random.default_rng(turn).random(rows).astype(np.float32)
        l.copy_(new)
        u.copy_(torch.from_numpy(nu))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        compare((tok.cpu().numpy(), prob.cpu().numpy(), kept.cpu().numpy()), new, nu, f"replay {turn}", **kw)
        ref = sample(new, nu, **kw)  # eager work between the replays
        assert np.array_equal(ref[0], tok.cpu().numpy())


def test_optional_outputs_and_host_form():
    rng = np.random.default_rng(9)
    l = (rng.normal(size=(5, 3000)) * 3).astype(np.float32)
    u = rng.random(5).astype(np.float32)
    got = ops.sample(l, u, temperature=0.8, top_k=[40, 0, 3, 100, 1], top_p=0.9, min_p=0.01)
    compare(got, l, u, "host", t=0.8, k=np.array([40, 0, 3, 100, 1]), p=0.9, mp=0.01)
    h = l.astype(np.float16)
    compare(ops.sample(h, u), h, u, "host fp16")
    assert all(a.shape == (0,) for a in ops.sample(l[:0], u[:0]))
    dl, du = torch.from_numpy(l).cuda(), torch.from_numpy(u).cuda()
    tok = torch.zeros(5, device="cuda", dtype=torch.int32)
    ws = torch.zeros(max(ops.sample_workspace_bytes(5, 3000), 256), device="cuda", dtype=torch.uint8)
    ops.sample_device(dl.data_ptr(), _native.F32, 5, 3000, du.data_ptr(), tok.data_ptr(), ws_ptr=ws.data_ptr(),
                      ws_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert np.array_equal(tok.cpu().numpy(), ops.sample(l, u)[0])


@pytest.mark.parametrize("compact", [False, True])
def test_next_token_is_the_mat_vec_and_the_sample(compact):
    rows, cols = 4096, 1024
    data = syn.matrix(syn.Q4_K, rows, cols, seed=10)
    t = ops.GgufTensor("output.weight", (cols, rows), syn.Q4_K, data.reshape(-1))
    if compact:
        t.prepare()
        t.compact()
    rng = np.random.default_rng(11)
    for i in range(6):
        x = rng.normal(size=cols).astype(np.float32)
        y = np.zeros(rows, np.float32)
        ops.mat_vec(t, x, y)
        kw = dict(temperature=(0.0, 5.0, 20.0)[i % 3], top_k=(0, 50)[i % 2], top_p=(1.0, 0.9)[i // 3], min_p=0.0)
        got = ops.next_token(t, x, float(np.float32(0.1 + 0.13 * i)), **kw)
        want = ops.sample(y[None], [np.float32(0.1 + 0.13 * i)], **kw)
        assert got == (want[0][0], want[1][0], want[2][0])
    with pytest.raises(ops.IllegalArgumentError):
        ops.next_token(t, x[:-1], 0.5)
    t.close()


# The ways a border is found: bins whose tokens fill the list, past it (the border's
# bin alone), a far bin of weight 0 (low temperatures), a min_p below the weights' unit,
# a top_k past the slabs, and the whole row by one workgroup.
WAYS = [dict(k=6000), dict(k=6000, t=0.05), dict(k=20000, t=0.03), dict(k=300, t=0.05, p=0.9), dict(k=64, t=0.02),
        dict(k=65), dict(k=2000, p=0.99, t=2.0), dict(k=2100, p=0.99, t=2.0), dict(k=2100, t=0.04, p=0.95),
        dict(mp=1e-15), dict(p=0.9, mp=1e-15), dict(k=30, mp=1e-15), dict(p=0.97, t=1.6), dict(p=0.999, t=4.0, mp=1e-3),
        dict(k=120000, p=0.95, t=1.5), dict(p=1e-9), dict(k=10**9, p=0.5)]


@pytest.mark.parametrize("i", range(len(WAYS)))
@pytest.mark.parametrize("vocab,rows,kind", [(128256, 3, _native.F32), (50257, 6, _native.BF16)])
def test_every_way_to_a_border(vocab, rows, kind, i):
    l = logits_of(rows, vocab, 100 + i, DTYPE[kind])
    u = np.random.default_rng(200 + i).random(rows).astype(np.float32)
    compare(sample(l, u, **WAYS[i]), l, u, f"{vocab} {WAYS[i]}", **WAYS[i])


@pytest.mark.parametrize("vocab", [262144, 300001, 4194304])
@pytest.mark.parametrize("kw", [dict(), dict(k=40, p=0.9), dict(p=0.9), dict(k=700, t=1.2), dict(mp=0.01)])
def test_large_vocabularies(vocab, kw):
    l = logits_of(2, vocab, vocab % 97)
    u = np.array([0.37, 0.93], np.float32)
    compare(sample(l, u, **kw), l, u, f"{vocab} {kw}", **kw)


def test_masks_of_the_lowest_value():
    """A mask written as the type's lowest finite value: tokens, of weight 0."""
    vocab = 40000
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        l = logits_of(4, vocab, 12).to(dtype)
        mask = torch.rand(4, vocab, generator=torch.Generator().manual_seed(1)) > 0.01
        l[mask.cuda()] = torch.finfo(dtype).min
        l[3] = torch.finfo(dtype).min
        u = np.array([0.1, 0.5, 0.9, 0.7], np.float32)
        for kw in (dict(), dict(k=50, p=0.9), dict(k=1000, p=0.9), dict(p=0.95), dict(mp=0.02), dict(k=900)):
            compare(sample(l, u, **kw), l, u, f"{dtype} {kw}", **kw)


def test_calls_on_two_streams_at_once():
    rows, vocab = 5, 60000
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = []
    for i, s in enumerate(side):
        l = logits_of(rows, vocab, 60 + i)
        u = torch.from_numpy(np.random.default_rng(i).random(rows).astype(np.float32)).cuda()
        p = torch.full((rows,), 0.9, device="cuda")
        out = [torch.zeros(rows, device="cuda", dtype=d) for d in (torch.int32, torch.float32, torch.int32)]
        ws = torch.zeros(ops.sample_workspace_bytes(rows, vocab), device="cuda", dtype=torch.uint8)
        runs.append((s, l, u, p, out, ws))
    torch.cuda.synchronize()
    for _ in range(6):
        for s, l, u, p, out, ws in runs:
            ops.sample_device(l.data_ptr(), _native.F32, rows, vocab, u.data_ptr(), out[0].data_ptr(),
                              top_p_ptr=p.data_ptr(), probs_ptr=out[1].data_ptr(), kept_ptr=out[2].data_ptr(),
                              ws_ptr=ws.data_ptr(), ws_bytes=ws.numel(), stream=s.cuda_stream)
    torch.cuda.synchronize()
    for _, l, u, _, out, _ in runs:
        compare([o.cpu().numpy() for o in out], l, u.cpu().numpy(), "two streams", p=0.9)


@pytest.mark.parametrize("vocab,stride", [(40001, 40003), (16384, 16385), (16385, 16388), (8192, 8192), (8193, 8200)])
def test_settings_of_their_own_over_long_rows(vocab, stride):
    rows = 24
    wide = logits_of(rows, stride, vocab)
    wide[:, vocab:] = 1e4  # behind the vocabulary: never read as a token
    rng = np.random.default_rng(vocab)
    kw = dict(t=rng.choice([0.0, 0.1, 0.6, 1.0, 1.7, 6.0], rows), k=rng.choice([0, 1, 7, 50, 64, 900, 3000, 10**6], rows),
              p=rng.choice([0.5, 0.9, 0.99, 1.0], rows), mp=rng.choice([0.0, 0.02, 0.3], rows))
    u = rng.random(rows).astype(np.float32)
    compare(sample(wide, u, vocab=vocab, **kw), wide[:, :vocab], u, "rows", **kw)


@pytest.mark.parametrize("vocab", [9000, 20000, 150000])
def test_crowds_of_equal_logits_at_the_border(vocab):
    """Hundreds of equal keys among the collected tokens: spread over the row, side by side, one ulp apart."""
    rng = np.random.default_rng(vocab)
    l = rng.normal(size=(6, vocab)).astype(np.float32) * 2.0
    l[0] = torch.from_numpy(l[0]).to(torch.bfloat16).float().numpy()
    l[1] = np.round(l[1])
    l[2, vocab // 3:vocab // 3 + 2000] = 9.5                      # neighbours
    l[3, rng.permutation(vocab)[:2500]] = 9.5
    l[3, rng.permutation(vocab)[:700]] = np.nextafter(np.float32(9.5), np.float32(10))
    l[4, rng.permutation(vocab)[:3000]] = 8.0                     # with others around them
    l[5, ::3] = 7.0
    l[5, 1:vocab:3] = 7.25
    dev = torch.from_numpy(l).cuda()
    u = rng.random(6).astype(np.float32)
    for kw in (dict(k=300), dict(k=1501, p=0.9003), dict(k=3333), dict(p=0.3007, t=1.2), dict(p=0.9501), dict(k=2600, mp=0.1)):
        compare(sample(dev, u, **kw), dev, u, f"crowds {kw}", **kw)
        half = dev.to(torch.bfloat16)
        compare(sample(half, u, **kw), half, u, f"crowds bf16 {kw}", **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_few_keys_on_both_sides_of_zero(dtype):
    tiny = 2.0**-130 if dtype is not torch.float16 else 2.0**-24  # (the types' subnormals)
    rng = np.random.default_rng(11)
    l = torch.from_numpy(rng.choice([-2 * tiny, -tiny, -0.0, 0.0, tiny, 2 * tiny], (3, 18000)).astype(np.float32)).to(dtype)
    dev = l.cuda()
    u = rng.random(3).astype(np.float32)
    for kw in (dict(k=2000), dict(k=3900), dict(k=9001, p=0.2003), dict(p=0.1507)):
        compare(sample(dev, u, **kw), dev, u, f"{dtype} {kw}", **kw)


def test_the_largest_batchs_workspace_serves_smaller_ones():
    vocab, most = 50257, 200  # (13 chunks a row: 200 rows are dealt to 10 parts, 150 and fewer to all 13)
    need = ops.sample_workspace_bytes(most, vocab)
    ws = torch.full((need,), 255, device="cuda", dtype=torch.uint8)
    l = logits_of(most, vocab, 70)
    u = torch.from_numpy(np.random.default_rng(71).random(most).astype(np.float32)).cuda()
    p = torch.full((most,), 0.9, device="cuda")
    out = [torch.zeros(most, device="cuda", dtype=d) for d in (torch.int32, torch.float32, torch.int32)]
    wants = None
    for rows in (most, 186, 171, 170, 157, 93, 33, 1):
        assert ops.sample_workspace_bytes(rows, vocab) <= need
        for o in out:
            o.fill_(-5)
        ops.sample_device(l.data_ptr(), _native.F32, rows, vocab, u.data_ptr(), out[0].data_ptr(), top_p_ptr=p.data_ptr(),
                          probs_ptr=out[1].data_ptr(), kept_ptr=out[2].data_ptr(), ws_ptr=ws.data_ptr(), ws_bytes=need,
                          stream=torch.cuda.current_stream().cuda_stream)
        got = [o.cpu().numpy() for o in out]
        if wants is None:
            compare([g[:9] for g in got], l[:9], u[:9].cpu().numpy(), "200 rows", p=0.9)
            wants = got
        assert all(np.array_equal(g[:rows], w[:rows]) and (g[rows:] == -5).all() for g, w in zip(got, wants)), rows


@pytest.mark.parametrize("vocab,rows", [(900, 40), (40000, 70)])
def test_results_in_the_place_of_their_settings(vocab, rows):
    l = logits_of(rows, vocab, 80)
    rng = np.random.default_rng(81)
    kw = dict(t=rng.choice([0.0, 0.7, 1.3], rows), k=rng.choice([0, 1, 40, 900], rows), p=rng.choice([0.8, 1.0], rows))
    u = rng.random(rows).astype(np.float32)
    t, p, du = (torch.from_numpy(np.asarray(a, np.float32)).cuda() for a in (kw["t"], kw["p"], u))
    k, kept = torch.from_numpy(kw["k"].astype(np.int32)).cuda(), torch.zeros(rows, device="cuda", dtype=torch.int32)
    ws = torch.zeros(max(ops.sample_workspace_bytes(rows, vocab), 256), device="cuda", dtype=torch.uint8)
    ops.sample_device(l.data_ptr(), _native.F32, rows, vocab, du.data_ptr(), k.data_ptr(), temperature_ptr=t.data_ptr(),
                      top_k_ptr=k.data_ptr(), top_p_ptr=p.data_ptr(), probs_ptr=du.data_ptr(), kept_ptr=kept.data_ptr(),
                      ws_ptr=ws.data_ptr(), ws_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    compare([a.cpu().numpy() for a in (k, du, kept)], l, u, "in place", **kw)


@pytest.mark.parametrize("vocab", [5000, 16384, 40000])
@pytest.mark.parametrize("kw", [dict(k=200, p=0.999), dict(k=1, p=0.9), dict(t=0.0, p=0.5), dict(k=2, p=0.99, mp=0.3),
                                dict(k=65, p=0.9999, t=3.0), dict(k=4500, p=0.99999), dict(k=3, p=0.7, t=float("inf"))])
def test_top_p_that_keeps_all_of_top_k_in_a_crowd(vocab, kw):
    """Thousands of equal logits through which top_k cuts; top_p then keeps every token that it left."""
    l = torch.full((4, vocab), -3.5, device="cuda")
    l[1, 100:103] = -3.0                     # the crowd is the second value
    l[2, ::7] = float("-inf")
    l[3, vocab // 2:] = float("-inf")
    l[3, :vocab // 2] = 0.0
    u = np.array([0.05, 0.9, 0.5, 0.99], np.float32)
    for dtype in (torch.float32, torch.bfloat16):
        compare(sample(l.to(dtype), u, **kw), l, u, f"crowd {vocab} {kw} {dtype}", **kw)


@pytest.mark.parametrize("kind", [syn.Q6_K, syn.Q8_0])
def test_next_token_of_a_long_vocabulary(kind):
    rows, cols = 20011, 512
    t = ops.GgufTensor("output.weight", (cols, rows), kind, syn.matrix(kind, rows, cols, seed=12).reshape(-1))
    rng = np.random.default_rng(13)
    for i in range(8):
        x = rng.normal(size=cols).astype(np.float32) * (0.0 if i == 7 else 1.0)  # (the last: equal logits)
        y = np.zeros(rows, np.float32)
        ops.mat_vec(t, x, y)
        kw = dict(temperature=(0.0, 5.0, 20.0, 1.0)[i % 4], top_k=(0, 50, 700)[i % 3], top_p=(1.0, 0.9)[i % 2], min_p=0.0)
        u = np.float32(0.07 + 0.12 * i)
        got = ops.next_token(t, x, float(u), **kw)
        host = ops.sample(y[None], [u], **kw)
        assert got == tuple(a[0] for a in host)
        compare(host, y[None], u, f"next token {kw}", t=kw["temperature"], k=kw["top_k"], p=kw["top_p"])
    t.close()
