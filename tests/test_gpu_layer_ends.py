"""Norms, rotary positions and appends at the ends of their ranges, on the GPU."""
import pytest
import torch

from gollek_amd import tensor_ops as ops
from tests import layer_ref as ref
from tests.layer_ref import BF16
from tests.test_gpu_layer_ops import close, ptr, stream, table

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
