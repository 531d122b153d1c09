"""Norms, rotary positions and the paged cache's append on the GPU against their
definitions in float64 (tests/layer_ref.py, where the tolerances are derived)."""
import numpy as np
import pytest
import torch

from gollek_amd import _native
from gollek_amd import tensor_ops as ops
from tests import layer_ref as ref
from tests.layer_ref import BF16, DTYPE, F16, F32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    ops.init(0)


def stream():
    return torch.cuda.current_stream().cuda_stream


def ptr(t):
    return 0 if t is None else t.data_ptr()


def rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape, sigma=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * sigma).to(dtype)


def close(got, want, off, type_id, what=""):
    got = got.detach().cpu().to(torch.float64)
    tol = off + ref.half_step(want, type_id) * (1 + 2.0**-10) + ref.half_step(off, type_id)
    bad = ~((got - want).abs() <= tol)
    worst = ((got - want).abs() / tol.clamp_min(1e-300)).max().item() if got.numel() else 0.0
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {worst:.3g} of what is allowed"


# ---- norms ------------------------------------------------------------------

def run_norm(rows, cols, x_type, hidden_type, y_type, *, post=False, gate=False, residual=True, weight=True, bias=False,
             hidden=True, y=True, layer=False, scale=1.0, eps=1e-6, pad=0, shift=0, seed=0, sigma=1.0):
    g = rng(seed)
    pitch = cols + pad

    def matrix(type_id, sigma=1.0):
        t = torch.full((rows * pitch + shift + 8,), float("nan"), dtype=DTYPE[type_id])
        v = t[shift:shift + rows * pitch].view(rows, pitch)[:, :cols]
        v.copy_(normal(g, rows, cols, sigma=sigma).to(DTYPE[type_id]))
        whole = t.cuda()
        return whole, whole[shift:shift + rows * pitch].view(rows, pitch)[:, :cols]

    xw, x = matrix(x_type, sigma)
    rw, r = matrix(hidden_type, 2.0) if residual else (None, None)
    hw, h = matrix(hidden_type) if hidden else (None, None)
    yw, yy = matrix(y_type) if y else (None, None)
    before = [None if w is None else w.clone() for w in (hw, yw)]
    vec = {n: normal(g, cols).cuda() if on else None for n, on in (("post", post), ("gate", gate), ("weight", weight), ("bias", bias))}
    print(f"[gpu] norm {rows}x{cols} x={x_type} hidden={hidden_type} y={y_type} layer={layer} pad={pad} shift={shift}", flush=True)
    stride = pitch if pad else 0
    ops.norm_device(ptr(x), x_type, rows, cols, x_stride=stride, post_weight_ptr=ptr(vec["post"]), gate_ptr=ptr(vec["gate"]),
                    scale=scale, residual_ptr=ptr(r), residual_stride=stride, hidden_ptr=ptr(h), hidden_type=hidden_type,
                    hidden_stride=stride, weight_ptr=ptr(vec["weight"]), bias_ptr=ptr(vec["bias"]),
                    kind=ops.NORM_LAYER if layer else ops.NORM_RMS, eps=eps, y_ptr=ptr(yy), y_type=y_type, y_stride=stride,
                    stream=stream())
    torch.cuda.synchronize()
    eh, ey, h_off, y_off = ref.norm(x, residual=r, layer=layer, scale=scale, eps=eps, **vec)
    if hidden:
        close(h, eh, h_off, hidden_type, "hidden")
    if y:
        close(yy, ey, y_off, y_type, "y")
    for whole, old, view in ((hw, before[0], h), (yw, before[1], yy)):  # nothing beside the rows
        if whole is not None:
            view.zero_()
            old[shift:shift + rows * pitch].view(rows, pitch)[:, :cols].zero_()
            assert torch.equal(torch.isnan(whole), torch.isnan(old))


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 8), (5, 63), (1, 64), (4, 100), (1, 257), (2, 1000), (7, 2880),
                                       (1, 4096), (33, 4096), (3, 5120), (2, 8191), (2, 14336), (1, 16384), (1, 16392),
                                       (2, 32768), (1, 65535), (1, 65536)])
@pytest.mark.parametrize("layer", [False, True])
def test_norm_sizes(rows, cols, layer):
    run_norm(rows, cols, BF16, F32, BF16, layer=layer, bias=layer, seed=cols)


@pytest.mark.parametrize("x_type", [F32, F16, BF16])
@pytest.mark.parametrize("hidden_type", [F32, F16, BF16])
@pytest.mark.parametrize("y_type", [F32, F16, BF16])
def test_norm_types(x_type, hidden_type, y_type):
    run_norm(3, 2048, x_type, hidden_type, y_type, post=True, gate=True, bias=True, scale=0.25, seed=3)
    run_norm(3, 999, x_type, hidden_type, y_type, post=True, layer=True, seed=4)


@pytest.mark.parametrize("kw", [dict(residual=False), dict(weight=False), dict(hidden=False), dict(y=False, post=True),
                                dict(post=True, gate=True, scale=-0.5), dict(gate=True), dict(scale=0.0), dict(eps=0.0),
                                dict(eps=1e-2, layer=True, post=True, bias=True), dict(residual=False, weight=False)])
def test_norm_parts(kw):
    run_norm(5, 640, F16, BF16, F32, seed=5, **kw)
    run_norm(2, 333, F16, BF16, F32, seed=6, **kw)


@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (0, 1), (8, 8), (16, 4), (5, 3)])
@pytest.mark.parametrize("cols", [512, 1001])
def test_norm_strides_and_alignment(pad, shift, cols):
    run_norm(6, cols, BF16, BF16, F16, pad=pad, shift=shift, seed=7)
    run_norm(6, cols, F32, F32, F32, pad=pad, shift=shift, post=True, seed=8)


def test_norm_of_many_rows():
    run_norm(70000, 24, BF16, BF16, BF16, seed=9)
    run_norm(2049, 768, BF16, BF16, BF16, post=True, seed=10)


def test_norm_large_and_small_values():
    run_norm(3, 4096, F32, F32, F32, sigma=1e15, seed=11)
    run_norm(3, 4096, F32, F32, F32, sigma=1e-12, residual=False, seed=12)
    run_norm(3, 4096, BF16, BF16, BF16, sigma=1e15, post=True, seed=13)


def test_norm_rows_of_zeros_and_infinities():
    x = torch.zeros(4, 96, device="cuda")
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3, 7] = 2.0
    h, y = torch.empty_like(x), torch.empty_like(x)
    ops.norm_device(ptr(x), F32, 4, 96, hidden_ptr=ptr(h), y_ptr=ptr(y), y_type=F32, eps=1e-6, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(h[[0, 1, 3]], x[[0, 1, 3]]) and torch.isnan(h[2, 5])
    assert torch.all(y[0] == 0) and torch.isnan(y[1, 3]) and torch.all(y[1, 4:] == 0) and torch.isnan(y[2]).all()
    assert abs(y[3, 7].item() - 2.0 / np.sqrt(4.0 / 96 + 1e-6)) < 1e-5 and torch.all(y[3, :7] == 0)


@pytest.mark.parametrize("cols", [2880, 77, 10000, 20001])
def test_norm_in_place(cols):
    g = rng(20)
    x, r = normal(g, 9, cols).cuda(), normal(g, 9, cols).cuda()
    w = normal(g, cols).cuda()
    eh, ey, h_off, y_off = ref.norm(x, residual=r, weight=w)
    ops.norm_device(ptr(x), F32, 9, cols, residual_ptr=ptr(r), hidden_ptr=ptr(r), weight_ptr=ptr(w), y_ptr=ptr(x),
                    y_type=F32, stream=stream())
    torch.cuda.synchronize()
    close(r, eh, h_off, F32, "hidden over its residual")
    close(x, ey, y_off, F32, "y over x")
    x = normal(g, 9, cols).cuda()
    eh, ey, h_off, y_off = ref.norm(x, post=w, layer=True)
    ops.norm_device(ptr(x), F32, 9, cols, post_weight_ptr=ptr(w), hidden_ptr=ptr(x), kind=ops.NORM_LAYER, stream=stream())
    torch.cuda.synchronize()
    close(x, eh, h_off, F32, "hidden over x")


def test_norm_of_column_ranges_of_one_matrix():
    g = rng(21)
    whole = normal(g, 5, 3 * 64).cuda()
    x = whole[:, :64].clone()
    ops.norm_device(ptr(whole), F32, 5, 64, x_stride=192, hidden_ptr=ptr(whole) + 64 * 4, hidden_stride=192,
                    y_ptr=ptr(whole) + 128 * 4, y_type=F32, y_stride=192, scale=0.5, stream=stream())
    torch.cuda.synchronize()
    eh, ey, h_off, y_off = ref.norm(x, scale=0.5)
    close(whole[:, 64:128], eh, h_off, F32)
    close(whole[:, 128:], ey, y_off, F32)
    assert torch.equal(whole[:, :64], x)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_host_norm(t):
    g = rng(22)
    x, r, w = normal(g, 4, 300).to(DTYPE[t]), normal(g, 4, 300).to(DTYPE[BF16]), normal(g, 300)
    host = x.view(torch.int16).numpy().view(np.uint16) if t == BF16 else x.numpy()
    h, y = ops.norm(host, w.numpy(), residual=r.view(torch.int16).numpy().view(np.uint16), y_type=F16, scale=2.0)
    eh, ey, h_off, y_off = ref.norm(x, residual=r, weight=w, scale=2.0)
    close(torch.from_numpy(h.view(np.int16)).view(torch.bfloat16), eh, h_off, BF16)
    close(torch.from_numpy(y), ey, y_off, F16)


# ---- rotary positions -------------------------------------------------------

def table(dims, base=10000.0, **kw):
    """The table's angles in float64 (its own definition is tested on the CPU)."""
    angles = base ** (-2.0 * np.arange(dims // 2) / dims)
    return ops.Rope(dims, base=base, **kw), angles


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("type_id", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,heads,dim,dims", [(1, 1, 2, 2), (1, 1, 64, 64), (3, 5, 128, 128), (7, 2, 80, 20),
                                                   (2, 3, 80, 80), (4, 2, 96, 48), (5, 1, 256, 64), (1, 3, 256, 256),
                                                   (2, 7, 72, 64), (3, 2, 66, 66), (2, 2, 250, 6), (333, 32, 64, 32),
                                                   (2, 65, 128, 128)])
def test_rope(tokens, heads, dim, dims, type_id, interleaved):
    g = rng(dim + dims)
    rope, angles = table(dims, layout=int(interleaved))
    x = normal(g, tokens, heads, dim).to(DTYPE[type_id]).cuda()
    at = torch.randint(0, 5000, (tokens,), generator=g, dtype=torch.int32).cuda()
    out = torch.full_like(x, float("nan"))
    print(f"[gpu] rope {tokens}x{heads}x{dim} dims={dims} type={type_id} interleaved={interleaved}", flush=True)
    rope.apply_device(ptr(x), type_id, tokens, heads, dim, ptr(at), ptr(out), stream=stream())
    torch.cuda.synchronize()
    want, off = ref.rotate(x, at, angles, 1.0, interleaved)
    close(out, want, off, type_id)
    assert torch.equal(out[..., dims:], x[..., dims:])
    rope.apply_device(ptr(x), type_id, tokens, heads, dim, ptr(at), ptr(x), stream=stream())  # in place
    torch.cuda.synchronize()
    assert torch.equal(x, out)
    rope.close()


def test_rope_far_and_negative_positions():
    g = rng(31)
    rope, angles = table(128, base=1000000.0)
    at = torch.tensor([0, 1, -1, 131071, 10**6, 2**24 + 1, 2**31 - 1, -(2**31)], dtype=torch.int32)
    x = normal(g, len(at), 2, 128).cuda()
    out = torch.empty_like(x)
    rope.apply_device(ptr(x), F32, len(at), 2, 128, ptr(at.cuda()), ptr(out), stream=stream())
    torch.cuda.synchronize()
    # 2^31 positions: float64 itself is off by 2^-53 * 2^31 radians
    want, off = ref.rotate(x, at, angles, 1.0, False)
    close(out, want, off + 2.0**-20 * (x.abs().cpu().double().amax()) * (at.abs().double() > 2**25)[:, None, None], F32)
    assert torch.equal(out[0], x[0])


@pytest.mark.parametrize("shift,pad", [(1, 0), (2, 4), (4, 3), (8, 8), (0, 1)])
@pytest.mark.parametrize("type_id", [F32, BF16])
def test_rope_strides_and_alignment(shift, pad, type_id):
    g = rng(32)
    tokens, heads, dim = 6, 3, 64
    pitch = heads * dim + pad
    rope, angles = table(dim)
    whole = torch.full((tokens * pitch + 16,), float("nan"), dtype=DTYPE[type_id], device="cuda")
    x = whole[shift:shift + tokens * pitch].view(tokens, pitch)[:, :heads * dim]
    x.copy_(normal(g, tokens, heads * dim))
    res = torch.full_like(whole, float("nan"))
    at = torch.arange(tokens, dtype=torch.int32).cuda() * 37
    rope.apply_device(ptr(x), type_id, tokens, heads, dim, ptr(at), ptr(res) + shift * whole.element_size(), x_stride=pitch,
                      out_stride=pitch, stream=stream())
    torch.cuda.synchronize()
    got = res[shift:shift + tokens * pitch].view(tokens, pitch)[:, :heads * dim].reshape(tokens, heads, dim)
    want, off = ref.rotate(x.reshape(tokens, heads, dim), at, angles, 1.0, False)
    close(got, want, off, type_id)
    assert int(torch.isnan(res).sum()) == res.numel() - tokens * heads * dim


def test_rope_scaled_tables_and_magnitude():
    g = rng(33)
    x = normal(g, 40, 4, 128)
    at = torch.arange(40, dtype=torch.int32) * 1000
    for kw in (dict(scaling=ops.ROPE_YARN, factor=4.0, original_context=8192.0, low=1.0, high=32.0),
               dict(scaling=ops.ROPE_LLAMA3, factor=8.0, original_context=8192.0, low=1.0, high=4.0),
               dict(scaling=ops.ROPE_LINEAR, factor=2.0, magnitude=0.75),
               dict(factors=np.linspace(1, 4, 64).astype(np.float32))):
        rope = ops.Rope(128, base=500000.0, **kw)
        f, magnitude = ops.rope_frequencies(128, base=500000.0, **kw)
        got = torch.from_numpy(rope.apply(x.numpy(), at.numpy()))
        # the frequencies come back in fp32: off by STEP of the angle, up to 40000 radians
        want, off = ref.rotate(x, at, f, magnitude, False)
        size = (x.abs().double()[..., :64] + x.abs().double()[..., 64:]).repeat(1, 1, 2)
        turn = at.double()[:, None, None] * torch.from_numpy(f).double().repeat(2)
        close(got, want, off + 2 * ref.STEP * magnitude * size * turn, F32)


@pytest.mark.parametrize("t", [F16, BF16])
def test_host_rope(t):
    g = rng(34)
    x = normal(g, 5, 3, 96).to(DTYPE[t])
    at = np.array([0, 3, 99, 1000, 65536], np.int32)
    rope, angles = table(48, layout=ops.ROPE_INTERLEAVED)
    got = rope.apply(x.view(torch.int16).numpy().view(np.uint16) if t == BF16 else x.numpy(), at)
    got = torch.from_numpy(got.view(np.int16)).view(DTYPE[t])
    want, off = ref.rotate(x, torch.from_numpy(at), angles, 1.0, True)
    close(got, want, off, t)
    with pytest.raises(ops.IllegalArgumentError):
        rope.apply(np.zeros((5, 3, 40), np.float32), at)  # heads shorter than what turns
    with pytest.raises(ops.IllegalArgumentError):
        rope.apply(np.zeros((5, 3, 96), np.float32), at[:4])


# ---- append -----------------------------------------------------------------

def run_append(tokens, q_heads, kv_heads, dim, type_id, cache_type, *, page=16, max_pages=8, positions=None, sequence=None,
               sequences=None, dims=None, interleaved=False, normed=False, rope=True, fused=True, in_place=False, table_edit=None,
               seed=0, pool=None):
    g = rng(seed)
    dims = dim if dims is None else dims
    sequences = tokens if sequences is None else sequences
    pool = sequences * max_pages + 3 if pool is None else pool
    pages = torch.randperm(pool, generator=g)[:sequences * max_pages].to(torch.int32).view(sequences, max_pages)
    if table_edit is not None:
        table_edit(pages)
    kc = normal(g, pool, kv_heads, page, dim).to(DTYPE[cache_type])
    vc = normal(g, pool, kv_heads, page, dim).to(DTYPE[cache_type])
    at = torch.randperm(max_pages * page, generator=g)[:tokens].to(torch.int32) if positions is None else positions
    seq = torch.arange(tokens, dtype=torch.int32) if sequence is None else sequence
    width = (q_heads + 2 * kv_heads) * dim
    src = normal(g, tokens, width, sigma=2.0).to(DTYPE[type_id])
    q, k, v = (s.unflatten(1, (-1, dim)) if s.numel() else s for s in src.split([q_heads * dim, kv_heads * dim, kv_heads * dim], 1))
    qn, kn = (1 + 0.3 * normal(g, dim), 1 + 0.3 * normal(g, dim)) if normed else (None, None)
    handle, angles = table(dims, layout=int(interleaved)) if rope else (None, np.zeros(0))
    dev = {n: (None if t is None else t.cuda()) for n, t in dict(src=src, kc=kc, vc=vc, pages=pages, at=at, qn=qn, kn=kn).items()}
    seq_dev = None if sequence is None else seq.cuda()
    size = dev["src"].element_size()
    if fused:
        where = [ptr(dev["src"]) + o * dim * size for o in (0, q_heads, q_heads + kv_heads)]
        parts, stride = [], width
    else:
        parts = [t.contiguous().cuda() for t in (q, k, v)]
        where, stride = [ptr(t) for t in parts], 0
    q_out = torch.full((tokens, q_heads, dim), float("nan"), dtype=DTYPE[cache_type], device="cuda")
    before = q_out.clone()
    cache = ops.KvCache(cache_type, ptr(dev["kc"]), ptr(dev["vc"]), pool, page, kv_heads, dim)
    print(f"[gpu] append {tokens} tokens {q_heads}/{kv_heads}x{dim} {type_id}->{cache_type} page={page} dims={dims} normed={normed}", flush=True)
    cache.append(where[1], where[2], type_id, tokens, ptr(dev["at"]), ptr(dev["pages"]), sequences, max_pages, rope=handle,
                 k_stride=stride, v_stride=stride, q_ptr=where[0] if q_heads else 0, q_heads=q_heads, q_stride=stride,
                 q_out_ptr=(where[0] if in_place else ptr(q_out)) if q_heads else 0, q_out_stride=stride if in_place else 0,
                 q_norm_ptr=ptr(dev["qn"]), k_norm_ptr=ptr(dev["kn"]), eps=1e-6, sequence_ptr=ptr(seq_dev), stream=stream())
    torch.cuda.synchronize()
    if in_place:
        q_out = dev["src"][:, :q_heads * dim].reshape(tokens, q_heads, dim)
        assert torch.equal(dev["src"][:, q_heads * dim:].cpu(), src[:, q_heads * dim:])
    live = [(t, int(seq[t]), int(at[t])) for t in range(tokens) if at[t] >= 0 and 0 <= seq[t] < sequences]
    mask = torch.zeros(tokens, dtype=torch.bool)
    mask[[t for t, _, _ in live]] = True

    def turned(h, weight):
        h, off = ref.f64(h), None
        if weight is not None:
            h, off = ref.head_norm(h, weight, 1e-6)
        return ref.rotate(h, at, angles, 1.0, interleaved, off)

    if q_heads:
        want, off = turned(q, qn)
        close(q_out[mask], want[mask], off[mask], cache_type, "q")
        if not in_place:
            assert torch.isnan(q_out[~mask]).all() and (before.numel() == q_out.numel())
    want, off = turned(k, kn)
    ek, ev = ref.f64(kc), ref.f64(vc)
    k_off = torch.zeros_like(ek)
    touched = torch.zeros(kc.shape[:3:2], dtype=torch.bool)
    for t, s, p in live:
        if p // page >= max_pages:
            continue
        number = int(pages[s, p // page])
        if not 0 <= number < pool:
            continue
        ek[number, :, p % page], ev[number, :, p % page] = want[t], ref.f64(v[t])
        k_off[number, :, p % page] = off[t]
        touched[number, p % page] = True
    got_k, got_v = dev["kc"].cpu(), dev["vc"].cpu()
    close(got_k, ek, k_off, cache_type, "k")
    close(got_v, ev, torch.zeros_like(ev), cache_type, "v")
    kept = ~touched[:, None, :].expand(kc.shape[:3])
    assert torch.equal(got_k[kept], kc[kept]) and torch.equal(got_v[kept], vc[kept])


@pytest.mark.parametrize("type_id", [F32, F16, BF16])
@pytest.mark.parametrize("cache_type", [F16, BF16])
@pytest.mark.parametrize("normed", [False, True])
def test_append_types(type_id, cache_type, normed):
    run_append(5, 8, 2, 128, type_id, cache_type, normed=normed, seed=40)
    run_append(3, 4, 4, 80, type_id, cache_type, normed=normed, dims=20, interleaved=True, seed=41)


@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,dims", [(1, 1, 1, 8, 8), (1, 32, 8, 128, 128), (2, 6, 2, 64, 32),
                                                              (9, 5, 5, 96, 96), (4, 16, 1, 256, 64), (3, 12, 4, 192, 192),
                                                              (64, 32, 4, 128, 128), (2, 7, 1, 72, 72), (1, 64, 64, 40, 10)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_shapes(tokens, q_heads, kv_heads, dim, dims, interleaved):
    run_append(tokens, q_heads, kv_heads, dim, BF16, BF16, dims=dims, interleaved=interleaved, normed=True, seed=dim)


@pytest.mark.parametrize("page", [16, 32, 128, 1024])
def test_append_page_sizes_and_prompts(page):
    # three sequences' tokens in one call: from 0, from the middle of a page, one token
    counts, starts = [70, 33, 1], [0, 21, 5]
    seq = torch.tensor(sum(([s] * n for s, n in enumerate(counts)), []), dtype=torch.int32)
    at = torch.cat([torch.arange(b, b + n) for b, n in zip(starts, counts)]).to(torch.int32)
    run_append(104, 8, 2, 64, BF16, F16, page=page, max_pages=max(1, 128 // page), positions=at, sequence=seq, sequences=3, seed=page)


def test_append_without_queries_rotation_or_fusion():
    run_append(6, 0, 2, 64, F32, BF16, seed=50)
    run_append(6, 4, 2, 64, F32, BF16, rope=False, seed=51)
    run_append(6, 4, 2, 64, F32, BF16, rope=False, normed=True, fused=False, seed=52)
    run_append(6, 4, 2, 64, F16, BF16, fused=False, seed=53)


def test_append_to_strided_queries():
    g = rng(58)
    tokens, heads, dim = 5, 4, 64
    k, v = (torch.zeros(6, 1, 16, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = ops.KvCache(BF16, ptr(k), ptr(v), 6, 16, 1, dim)
    src = normal(g, tokens, heads + 2, dim).cuda()
    at, pages = torch.arange(tokens, dtype=torch.int32).cuda(), torch.arange(5, dtype=torch.int32).cuda()
    out = torch.full((tokens * 301 + 8,), float("nan"), dtype=torch.bfloat16, device="cuda")
    rope, angles = table(dim)
    stride = (heads + 2) * dim
    cache.append(ptr(src) + heads * dim * 4, ptr(src) + (heads + 1) * dim * 4, F32, tokens, ptr(at), ptr(pages), 5, 1, rope=rope,
                 k_stride=stride, v_stride=stride, q_ptr=ptr(src), q_heads=heads, q_stride=stride, q_out_ptr=ptr(out) + 6,
                 q_out_stride=301, stream=stream())
    torch.cuda.synchronize()
    rows = out[3:3 + tokens * 301].view(tokens, 301)
    want, off = ref.rotate(src[:, :heads], at, angles, 1.0, False)
    close(rows[:, :heads * dim].reshape(tokens, heads, dim), want, off, BF16)
    assert int(torch.isnan(out).sum()) == out.numel() - tokens * heads * dim


@pytest.mark.parametrize("type_id", [F16, BF16])
def test_append_queries_in_place(type_id):
    run_append(6, 4, 2, 64, type_id, BF16 if type_id == BF16 else F16, in_place=True, normed=True, seed=54)


def test_append_padding_bad_pages_and_places_past_the_table():
    at = torch.tensor([3, -1, 17, -(2**31), 127, 128, 2**31 - 1, 40, 41, 60], dtype=torch.int32)
    seq = torch.tensor([0, 1, 2, 3, 4, 5, 6, -1, 12, 2**31 - 1], dtype=torch.int32)

    def edit(pages):
        pages[2, 1] = -1      # token 2's page
        pages[4, 7] = 2**30   # token 4's

    run_append(10, 4, 2, 64, F32, BF16, positions=at, sequence=seq, sequences=12, table_edit=edit, seed=55)


def test_append_to_a_cache_past_32_bits():
    # 2^32 + elements: 9 GB of keys and as much of values
    kv_heads, page, dim = 8, 16, 128
    pool = (2**32) // (kv_heads * page * dim) + 2
    k, v = (torch.empty(pool, kv_heads, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k[-1], v[-1], k[0], v[0] = 0, 0, 0, 0
    g = rng(56)
    src = normal(g, 1, 3 * kv_heads, dim).cuda()
    at, pages = torch.tensor([5], dtype=torch.int32).cuda(), torch.tensor([[pool - 1]], dtype=torch.int32).cuda()
    cache = ops.KvCache(BF16, ptr(k), ptr(v), pool, page, kv_heads, dim)
    q = torch.empty(1, kv_heads, dim, dtype=torch.bfloat16, device="cuda")
    cache.append(ptr(src) + kv_heads * dim * 4, ptr(src) + 2 * kv_heads * dim * 4, F32, 1, ptr(at), ptr(pages), 1, 1,
                 q_ptr=ptr(src), q_heads=kv_heads, q_out_ptr=ptr(q), stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(k[-1, :, 5], src[0, kv_heads:2 * kv_heads].bfloat16()) and torch.equal(v[-1, :, 5], src[0, 2 * kv_heads:].bfloat16())
    assert not k[0].any() and not v[0].any() and not k[-1, :, :5].any() and not k[-1, :, 6:].any()
    lengths = torch.tensor([6], dtype=torch.int32).cuda()
    out = torch.empty(1, kv_heads, dim, device="cuda")
    ws = torch.empty(max(256, cache.attend_workspace_bytes(1, kv_heads, 1)), dtype=torch.uint8, device="cuda")
    cache.attend(ptr(q), 1, kv_heads, ptr(lengths), ptr(pages), 1, ptr(out), F32, scale=ref.softmax_scale(dim), ws_ptr=ptr(ws),
                 ws_bytes=ws.numel(), stream=stream())
    torch.cuda.synchronize()
    want, off = ref.attention(q[0], k[-1, :, :6].transpose(0, 1), v[-1, :, :6].transpose(0, 1), scale=ref.softmax_scale(dim))
    close(out[0], want, off, F32)


def test_append_and_rope_on_another_stream_and_captured():
    g = rng(57)
    tokens, kv_heads, dim, page = 4, 2, 64, 16
    k, v = (torch.zeros(9, kv_heads, page, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    pages = torch.randperm(8, generator=g).to(torch.int32).view(4, 2).cuda()
    src = torch.zeros(tokens, 3 * kv_heads, dim, device="cuda")
    at = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    q = torch.zeros(tokens, kv_heads, dim, dtype=torch.float16, device="cuda")
    rope, angles = table(dim)
    cache = ops.KvCache(F16, ptr(k), ptr(v), 9, page, kv_heads, dim)
    size, stride = kv_heads * dim * 4, 3 * kv_heads * dim

    def call(s):
        cache.append(ptr(src) + size, ptr(src) + 2 * size, F32, tokens, ptr(at), ptr(pages), 4, 2, rope=rope, k_stride=stride,
                     v_stride=stride, q_ptr=ptr(src), q_heads=kv_heads, q_stride=stride, q_out_ptr=ptr(q), stream=s)

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(side.cuda_stream)
    for step in range(4):  # replays with other inputs, eager work between
        src.copy_(normal(g, tokens, 3 * kv_heads, dim))
        at.copy_(torch.randint(0, 32, (tokens,), generator=g, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = (q.clone(), k.clone(), v.clone())
        k.zero_(), v.zero_(), q.zero_()
        with torch.cuda.stream(side):
            call(side.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(got[0], q)
        want, off = ref.rotate(src[:, :kv_heads], at, angles, 1.0, False)
        close(q, want, off, F16)
        for t in range(tokens):
            number, slot = int(pages[t, int(at[t]) // page]), int(at[t]) % page
            assert torch.equal(got[1][number, :, slot], k[number, :, slot]) and torch.equal(got[2][number, :, slot], v[number, :, slot])
            assert k[number, :, slot].any()
