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
