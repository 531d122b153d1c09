"""Norms, rotary positions, appends and attention at the ends of their ranges, on the GPU."""
import numpy as np
import pytest
import torch

from gollek_amd import tensor_ops as ops
from tests import layer_ref as ref
from tests.layer_ref import BF16, F16, F32
from tests.test_gpu_layer_ops import close, ptr, run_norm, stream, table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    ops.init(0)


def rope_of_many_tokens(tokens):
    """One head of one pair a token: against float64 at both ends, in between against calls of fewer tokens."""
    rope, angles = table(2)
    at = (torch.arange(tokens, device="cuda", dtype=torch.int32) * 7) % 5003
    x = ((torch.arange(2 * tokens, device="cuda", dtype=torch.int32) * 13 % 1001).to(torch.float32) / 250 - 2).bfloat16()
    out, parts = torch.full_like(x, float("nan")), torch.full_like(x, float("nan"))
    print(f"[gpu] rope {tokens} tokens", flush=True)
    rope.apply_device(ptr(x), BF16, tokens, 1, 2, ptr(at), ptr(out), stream=stream())
    for first in range(0, tokens, 1 << 22):
        n = min(1 << 22, tokens - first)
        rope.apply_device(ptr(x) + 4 * first, BF16, n, 1, 2, ptr(at) + 4 * first, ptr(parts) + 4 * first, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(out, parts)
    for s in (slice(0, 1000), slice(tokens - 1000, tokens)):
        want, off = ref.rotate(x.view(tokens, 1, 2)[s], at[s], angles, 1.0, False)
        close(out.view(tokens, 1, 2)[s], want, off, BF16)


def test_rope_whose_surplus_waves_would_count_past_32_bits():
    # 64 heads a wave: the waves behind the last token would be at head 64 * 2^25
    rope_of_many_tokens((1 << 25) + 1)


def test_rope_of_more_tokens_than_one_grid():
    rope_of_many_tokens((1 << 26) + 5)


@pytest.mark.parametrize("numbered", [False, True])
def test_append_of_more_tokens_than_one_grid(numbered):
    # a place for a few tokens around the borders of launches; the others' pages are none
    tokens, page, dim = (1 << 26) + 5, 16, 8
    chosen = [0, 1, (1 << 25) - 1, 1 << 25, (1 << 25) + 1, (1 << 26) - 1, 1 << 26, tokens - 1]
    k, v = (torch.full((len(chosen) + 1, 1, page, dim), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    pages = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(tokens, device="cuda", dtype=torch.int32) % page
    sequence = torch.arange(tokens, device="cuda", dtype=torch.int32).flip(0) if numbered else None
    for i, t in enumerate(chosen):
        pages[tokens - 1 - t if numbered else t] = i
    src = (torch.arange(tokens * dim, device="cuda", dtype=torch.int32) * 31 % 2039).to(torch.float16).view(tokens, dim)
    q_out = torch.full_like(src, float("nan"))
    cache = ops.KvCache(F16, ptr(k), ptr(v), len(chosen) + 1, page, 1, dim)
    print(f"[gpu] append {tokens} tokens, numbered={numbered}", flush=True)
    cache.append(ptr(src), ptr(src), F16, tokens, ptr(at), ptr(pages), tokens, 1, q_ptr=ptr(src), q_heads=1, q_out_ptr=ptr(q_out),
                 sequence_ptr=ptr(sequence), stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(q_out, src)
    want = torch.full_like(k, 9.0)
    for i, t in enumerate(chosen):
        want[i, 0, t % page] = src[t]
    assert torch.equal(k, want) and torch.equal(v, want)


@pytest.mark.parametrize("sequences,heads,max_pages", [(256, 65535, 200), (4095, 4097, 20), (255, 65535, 1)])
def test_attention_of_almost_2_to_24_rows(sequences, heads, max_pages):
    # one token each: its value, whatever the score
    page, dim = 16, 8
    k = torch.ones(3, heads, page, dim, dtype=torch.float16, device="cuda")
    v = torch.randn(3, heads, page, dim, dtype=torch.float16, device="cuda")
    q = torch.ones(sequences, heads, dim, dtype=torch.float16, device="cuda")
    pages = torch.full((sequences, max_pages), -1, dtype=torch.int32, device="cuda")
    pages[:, 0] = torch.arange(sequences, device="cuda") % 3
    lengths = torch.ones(sequences, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, float("nan"))
    cache = ops.KvCache(F16, ptr(k), ptr(v), 3, page, heads, dim)
    need = cache.attend_workspace_bytes(sequences, heads, max_pages)
    ws = torch.zeros(max(need, 256), dtype=torch.uint8, device="cuda")
    print(f"[gpu] attend {sequences} x {heads}, table of {max_pages}, workspace {need}", flush=True)
    cache.attend(ptr(q), sequences, heads, ptr(lengths), ptr(pages), max_pages, ptr(out), F16, scale=1.0, ws_ptr=ptr(ws),
                 ws_bytes=need, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(out, v[pages[:, 0].long(), :, 0])


@pytest.mark.parametrize("cols,sigma", [(64, 1.5e18), (4096, 2.6e17), (8000, 1.9e17), (65536, 7e16)])
@pytest.mark.parametrize("post", [False, True])
def test_norm_of_rows_near_the_largest(cols, sigma, post):
    # root mean squares a little below 1.8e19 / sqrt(cols) (64: a third below, rows of so few vary)
    run_norm(5, cols, F32, F32, F32, sigma=sigma, post=post, seed=80)


@pytest.mark.parametrize("sigma", [1e-15, 1e-18])
def test_norm_of_small_rows_without_eps(sigma):
    run_norm(5, 1000, F32, F32, F32, sigma=sigma, residual=False, eps=0.0, seed=81)


def test_a_table_closed_while_a_stream_is_captured():
    # as the garbage collector may: the capture goes on, with the table that it holds
    rope, _ = table(64)
    other, _ = table(64, base=5000.0)
    x = torch.randn(4, 2, 64, device="cuda")
    at = torch.arange(4, dtype=torch.int32, device="cuda")
    want, out = torch.empty_like(x), torch.zeros_like(x)
    rope.apply_device(ptr(x), F32, 4, 2, 64, ptr(at), ptr(want), stream=stream())
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        rope.apply_device(ptr(x), F32, 4, 2, 64, ptr(at), ptr(out), stream=side.cuda_stream)
        other.close()
        twice = out * 2
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(twice, 2 * want)


@pytest.mark.parametrize("first", [0, 100000])
def test_rope_sines_next_to_half_a_revolution(first):
    # (0, 1) becomes (-sin, cos): each off by no more than 8 half steps of itself (sine and cosine 4
    # ulp, and a product), small ones too, besides what position * frequency is off by in 64 bits:
    # three roundings of the angle in revolutions, 2^-53 each
    rope, angles = table(128)
    tokens = 4096
    at = first + torch.arange(tokens, dtype=torch.int32)
    x = torch.cat([torch.zeros(tokens, 64), torch.ones(tokens, 64)], 1).cuda()
    out = torch.empty_like(x)
    rope.apply_device(ptr(x), F32, tokens, 1, 128, ptr(at.cuda()), ptr(out), stream=stream())
    torch.cuda.synchronize()
    t = at.numpy()[:, None].astype(np.longdouble) * (np.longdouble(10000) ** (-2 * np.arange(64, dtype=np.longdouble) / 128))
    want = torch.from_numpy(np.concatenate([-np.sin(t), np.cos(t)], 1).astype(np.float64))
    off = 8 * ref.STEP * want.abs() + 4 * 2.0**-53 * torch.from_numpy(np.concatenate([t, t], 1).astype(np.float64)) + 1e-30
    bad = (out.cpu().double() - want).abs() > off
    assert not bad.any(), (int(bad.sum()), want[bad][:4], out.cpu()[bad][:4])
