"""What an attention's numbers keep of fp32, on the GPU: results of every type against the
definition in float64, with tolerances that count roundings of fp32 alone, and values and
settings at the ends of their types."""
import pytest
import torch

from gollek_amd import tensor_ops as ops
from tests import layer_ref as ref
from tests.layer_ref import BF16, DTYPE, F16, F32, STEP
from tests.test_gpu_attention import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    ops.init(0)


def rows_of(b, s):
    """Keys and values (tokens, kv_heads, dim) of sequence s."""
    length = b.lengths[s]
    begin = max(0, length - b.window) if b.window else 0
    return ref.gather(b.k, b.table[s], length, begin), ref.gather(b.v, b.table[s], length, begin)


def definition(q, k, v, scale, softcap=0.0, sinks=None):
    """One sequence in float64, and how far a computation in fp32 may be from it before the
    result's own rounding.  On a score (dim + 8) STEP of scale |q| . |k| for its sum in any
    order, and 4 STEP of it for the scaling; a cap keeps it to 16 STEP of the capped score
    (quotient, tanh and product, each relative to their own result).  A weight is off by
    twice the most of these (its own and the largest one's), and by 16 STEP for its
    exponential, the pieces it is multiplied in (2^-23) and the quotient; sums of n terms in
    any order add n STEP of the sum of magnitudes."""
    q, k, v = ref.f64(q), ref.f64(k), ref.f64(v)
    group = q.shape[0] // k.shape[1]
    kk, vv = k.transpose(0, 1).repeat_interleave(group, 0), v.transpose(0, 1).repeat_interleave(group, 0)
    s = scale * torch.bmm(kk, q[:, :, None])[:, :, 0]
    near = (q.shape[1] + 8) * STEP * abs(scale) * torch.bmm(kk.abs(), q.abs()[:, :, None])[:, :, 0] + 4 * STEP * s.abs()
    if softcap:
        s = softcap * torch.tanh(s / softcap)
        near = near + 16 * STEP * s.abs()
    top = s.amax(1, keepdim=True)
    if sinks is not None:
        sinks = ref.f64(sinks)[:, None]
        top = torch.maximum(top, sinks)
    p = torch.exp(s - top)
    total = p.sum(1, keepdim=True) + (torch.exp(sinks - top) if sinks is not None else 0.0)
    p = p / total
    size = torch.bmm(p[:, None, :], vv.abs())[:, 0]
    return torch.bmm(p[:, None, :], vv)[:, 0], (2 * near.amax(1, keepdim=True) + (k.shape[0] + 16) * STEP) * size


def between(got, want, off, out_type, what):
    """Rounding keeps order: an fp32 number no further than off from want becomes one between
    the roundings of want - off and want + off."""
    got = got.detach().cpu().to(torch.float64)
    low, high = ((want + d).to(torch.float32).to(DTYPE[out_type]).to(torch.float64) for d in (-off, off))
    bad = ~((low <= got) & (got <= high))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, {got[bad][:3]} for {want[bad][:3]}"


def compare(b, out, out_type, rows=None, *, scale=None, softcap=0.0, sinks=None):
    scale = ref.softmax_scale(b.dim) if scale is None else scale
    torch.cuda.synchronize()
    for s in range(len(b.lengths)) if rows is None else rows:
        want, off = definition(b.q[s], *rows_of(b, s), scale, softcap, sinks)
        between(out[s], want, off, out_type, f"sequence {s} of length {b.lengths[s]}")


@pytest.mark.parametrize("out_type", [F16, BF16, F32])
@pytest.mark.parametrize("cache_type", [F16, BF16])
@pytest.mark.parametrize("kv_heads", [1, 8])
def test_weights_keep_fp32(cache_type, out_type, kv_heads):
    # few tokens of almost equal weight: nothing but the weights' own pieces is off by much;
    # among 60000 results some lie next to a border between two numbers of the type
    b = Batch([8, 5, 7, 8, 6] * 24, 8, kv_heads, 64, cache_type, q_sigma=0.02, seed=50 + kv_heads)
    compare(b, b.attend(out_type), out_type)


@pytest.mark.parametrize("softcap", [0.5, 50.0, 1e3, 1e5, 1e8, 1e15])
@pytest.mark.parametrize("out_type", [F16, BF16, F32])
@pytest.mark.parametrize("cache_type", [F16, BF16])
def test_a_cap_of_any_size(cache_type, out_type, softcap):
    # a cap far above every score is none; a workgroup a head, a wave a head, a chunk of many
    b = Batch([0, 1, 77, 400, 3000], 8, 2, 128, cache_type, seed=60)
    compare(b, b.attend(out_type, softcap=softcap), out_type, [1, 2, 3, 4], softcap=softcap)
    b = Batch([(11 * i) % 50 + 1 for i in range(500)], 8, 4, 64, cache_type, seed=61)
    compare(b, b.attend(out_type, softcap=softcap), out_type, range(0, 500, 71), softcap=softcap)


def test_a_cap_far_above_every_score_changes_nothing():
    b = Batch([77, 2000], 8, 2, 64, BF16, seed=62)
    for out_type in (F16, BF16):
        bits = [b.attend(out_type, softcap=c).float() for c in (0.0, 1e9)]
        assert torch.allclose(*bits, rtol=2 * torch.finfo(DTYPE[out_type]).eps, atol=1e-6)


INF, NAN = float("inf"), float("nan")


def poke(b, s, position, head, dim, value):
    """A value of sequence s's token at `position`."""
    b.v[int(b.table[s, position // b.page]), head, position % b.page, dim] = value


@pytest.mark.parametrize("lengths,kv_heads,dim,window", [
    ([1, 40, 700, 90, 33], 2, 128, 0),                        # a workgroup a head
    ([1, 40, 20000, 90, 9000], 2, 64, 0),                     # cut into chunks, some joined by many
    ([1, 40, 6000] + [90] * 300, 2, 64, 0),                   # by few
    ([1, 40, 100, 90, 33] + [60] * 300, 8, 80, 0),            # a wave a head
    ([1, 40, 100, 90, 33] + [60] * 300, 4, 256, 0),
    ([1, 40, 3000, 90, 33], 2, 192, 50)])
@pytest.mark.parametrize("cache_type,out_type", [(F16, F32), (F16, BF16), (BF16, F32), (BF16, F16), (F16, F16)])
@pytest.mark.parametrize("with_sinks", [False, True])
def test_infinite_values(lengths, kv_heads, dim, window, cache_type, out_type, with_sinks):
    # an infinite value makes its dim infinite, also where its weight is tiny; two of other
    # signs, or a NaN, make it NaN; every other dim, head and sequence stays as it was
    b = Batch(lengths, 2 * kv_heads, kv_heads, dim, cache_type, window=window, q_sigma=1.0, seed=70)
    sinks = torch.linspace(-3, 3, 2 * kv_heads).cuda() if with_sinks else None
    clean = b.device().attend(F32, sinks=sinks).cpu()
    last = lengths[2] - 1
    poke(b, 0, 0, 1, 3, INF)           # the only token
    poke(b, 1, 39, 0, 0, -INF)
    poke(b, 1, 12, 1, dim - 1, INF)
    poke(b, 2, last, 0, 5, INF)
    poke(b, 2, last - 30, 0, 5, INF)   # twice
    poke(b, 2, last - 7, 0, 6, INF)
    poke(b, 2, last - 48, 0, 6, -INF)  # both signs
    poke(b, 2, last - 9, 1, 7, NAN)
    poke(b, 2, last - 9, 1, 8, NAN)
    poke(b, 2, last - 20, 1, 8, INF)   # and one with a NaN
    want = {(0, 1, 3): INF, (1, 0, 0): -INF, (1, 1, dim - 1): INF, (2, 0, 5): INF, (2, 0, 6): NAN, (2, 1, 7): NAN, (2, 1, 8): NAN}
    out = b.device().attend(out_type, sinks=sinks).cpu().float()
    for (s, head, d), value in want.items():
        got = out[s, 2 * head:2 * head + 2, d]
        assert torch.isnan(got).all() if value != value else (got == value).all(), (s, head, d, got)
        out[s, 2 * head:2 * head + 2, d] = clean[s, 2 * head:2 * head + 2, d]
    eps = torch.finfo(DTYPE[out_type]).eps
    assert torch.allclose(out, clean, rtol=eps, atol=2e-6 if out_type != F16 else 1e-5)


@pytest.mark.parametrize("cache_type", [F16, BF16])
@pytest.mark.parametrize("lengths", [[300], [20000], [300] + [40] * 600])
def test_infinite_values_of_no_weight_to_speak_of(lengths, cache_type):
    # their token's weight is e^-200: far below what fp32 holds, and above nothing
    b = Batch(lengths, 4, 2, 64, cache_type, seed=71)
    b.q[0].fill_(1.0)
    for position in range(lengths[0]):
        b.k[int(b.table[0, position // 16]), :, position % 16] = 0.0
    for position in (7, lengths[0] - 2):
        b.k[int(b.table[0, position // 16]), :, position % 16] = -200.0 / 64
        poke(b, 0, position, 0, 9, -INF)
    out = b.device().attend(F32, scale=1.0).cpu()
    assert (out[0, :2, 9] == -INF).all()
    out[0, :2, 9] = 0.0
    assert torch.isfinite(out).all()


def test_infinite_values_outside_a_window_or_a_length():
    b = Batch([100, 100, 100], 4, 2, 64, F16, seed=72, window=40)
    want = b.attend(F32).cpu()
    inside = torch.zeros(b.v.shape[0], 16, dtype=torch.bool)
    for s in range(3):
        for position in range(60, 100):
            inside[int(b.table[s, position // 16]), position % 16] = True
    b.v.masked_fill_(~inside[:, None, :, None], INF)
    assert torch.equal(b.device().attend(F32).cpu(), want)


@pytest.mark.parametrize("lengths", [[0, 1, 77, 400], [0, 1, 77, 9000], [5, 60] * 300])
def test_sinks_at_the_ends(lengths):
    # a sink past every score takes all weight, one at the lowest value none, and a NaN is its head's
    b = Batch(lengths, 8, 4, 64, BF16, seed=63)
    most = torch.finfo(torch.float32).max
    sinks = torch.tensor([most, 3e38, INF, -most, -INF, NAN, 0.5, -3e38]).cuda()
    out, plain = b.attend(F32, sinks=sinks).cpu(), b.attend(F32).cpu()
    assert not out[:, :3].any()
    assert torch.equal(out[:, [3, 4, 7]], plain[:, [3, 4, 7]])
    some = [i for i, n in enumerate(lengths) if n > 0]
    assert torch.isnan(out[some, 5]).all()
    for s in range(4):
        if lengths[s]:
            want, off = definition(b.q[s], *rows_of(b, s), ref.softmax_scale(64), 0.0, torch.full((8,), 0.5))
            between(out[s, 6], want[6], off[6], F32, f"sequence {s}")


def test_large_values_under_growing_scores():
    # a score up to 2^8 above those before it: its weight and bf16's largest values stay in range
    b = Batch([1000], 2, 1, 64, BF16, seed=64)
    b.q.fill_(1.0)
    b.v.fill_(1.0)
    for position in range(1000):
        b.k[int(b.table[0, position // 16]), 0, position % 16] = 0.0 if position % 640 < 600 else 5.0 / 64
        if position % 640 == 639:
            b.v[int(b.table[0, position // 16]), 0, position % 16] = 3e36 * torch.linspace(-1, 1, 64)
    b.device()
    compare(b, b.attend(F32, scale=1.0), F32, scale=1.0)


@pytest.mark.parametrize("lengths,some", [([3000], True), ([900] * 5, False)])
def test_a_workspace_one_byte_short_is_refused(lengths, some):
    # tables of up to 32 tiles of 32 tokens (heads of 64, few of them) are not cut and need none: 900
    # tokens' 57 pages are 29 tiles
    b = Batch(lengths, 4, 2, 64, BF16, seed=65)
    assert (b.need > 0) == some
    if some:
        b.need -= 1
        with pytest.raises(ops.IllegalArgumentError, match="Workspace"):
            b.attend(F32)
        b.need += 1
    compare(b, b.attend(F32), F32)
    assert torch.all(b.ws[b.need:] == 0xFF)
