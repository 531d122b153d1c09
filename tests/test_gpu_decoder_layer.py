"""A decoder layer's attention block as it would run: the norm, the fused q / k / v
product, the new keys and values into the paged cache with their rotation, attention, the
output product onto the residual stream and the norm behind it.  A prompt of ragged
sequences goes in first (its tokens as rows of growing lengths), then decoded tokens,
eagerly and as one captured graph.  Every stage is checked against float64 on the inputs
that it had."""
import numpy as np
import pytest
import torch

from gollek_amd import _native
from gollek_amd import synthetic as syn
from gollek_amd import tensor_ops as ops
from tests import layer_ref as ref
from tests.layer_ref import BF16, DTYPE, F32
from tests.test_gpu_layer_ops import close, normal, ptr, rng
from tests.test_gpu_linear import Weight, check, expected

pytestmark = pytest.mark.gpu

H, QH, KV, D, PAGE, PAGES = 512, 8, 2, 64, 16, 12
PROMPTS = [37, 1, 90, 16]
BASE = 10000.0


class Layer:
    def __init__(self, kind, cache_type, most, seed):
        self.qkv = Weight(kind, (QH + 2 * KV) * D, H, seed)
        self.out = Weight(kind, H, QH * D, seed + 1)
        g = self.g = rng(seed)
        n = len(PROMPTS)
        self.pre, self.post = (1 + 0.2 * normal(g, H)).cuda(), (1 + 0.2 * normal(g, H)).cuda()
        self.gate = (0.3 * normal(g, H)).cuda()
        self.qn, self.kn = (1 + 0.2 * normal(g, D)).cuda(), (1 + 0.2 * normal(g, D)).cuda()
        dtype = DTYPE[cache_type]
        self.type = cache_type
        self.k, self.v = (torch.full((n * PAGES + 1, KV, PAGE, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        self.table = torch.randperm(n * PAGES, generator=g).to(torch.int32).view(n, PAGES).cuda()
        self.cache = ops.KvCache(cache_type, ptr(self.k), ptr(self.v), n * PAGES + 1, PAGE, KV, D)
        self.rope = ops.Rope(D, base=BASE)
        z = lambda *s, d=torch.float32: torch.zeros(s, device="cuda", dtype=d)  # noqa: E731
        self.stream, self.x = z(most, H), z(most, H, d=torch.bfloat16)
        self.heads, self.q = z(most, (QH + 2 * KV) * D), z(most, QH, D, d=dtype)
        self.attn, self.block = z(most, QH * D, d=torch.bfloat16), z(most, H)
        self.after, self.y = z(most, H), z(most, H, d=torch.bfloat16)
        self.positions, self.sequence, self.lengths = (z(most, d=torch.int32) for _ in range(3))
        self.rows = torch.zeros(most, PAGES, dtype=torch.int32, device="cuda")
        need = max(w.handle.linear_workspace_bytes(m) for w in (self.qkv, self.out) for m in range(1, most + 1))
        need = max(need, self.cache.attend_workspace_bytes(most, QH, PAGES))
        self.ws = torch.zeros(max(need, 256), dtype=torch.uint8, device="cuda")

    def inputs(self, tokens):
        """tokens: (sequence, position) of each row."""
        m = len(tokens)
        self.stream[:m].copy_(normal(self.g, m, H, sigma=2.0))
        self.sequence[:m].copy_(torch.tensor([s for s, _ in tokens], dtype=torch.int32))
        self.positions[:m].copy_(torch.tensor([p for _, p in tokens], dtype=torch.int32))
        self.lengths[:m].copy_(torch.tensor([p + 1 for _, p in tokens], dtype=torch.int32))
        self.rows[:m].copy_(self.table[[s for s, _ in tokens]])
        torch.cuda.synchronize()

    def run(self, m, stream):
        width, size = (QH + 2 * KV) * D, 4
        ws = dict(ws_ptr=ptr(self.ws), ws_bytes=self.ws.numel(), stream=stream)
        ops.norm_device(ptr(self.stream), F32, m, H, weight_ptr=ptr(self.pre), y_ptr=ptr(self.x), y_type=BF16, stream=stream)
        self.qkv.handle.linear(ptr(self.x), m, ptr(self.heads), F32, **ws)
        self.cache.append(ptr(self.heads) + QH * D * size, ptr(self.heads) + (QH + KV) * D * size, F32, m,
                          ptr(self.positions), ptr(self.table), len(PROMPTS), PAGES, rope=self.rope, k_stride=width,
                          v_stride=width, q_ptr=ptr(self.heads), q_heads=QH, q_stride=width, q_out_ptr=ptr(self.q),
                          q_norm_ptr=ptr(self.qn), k_norm_ptr=ptr(self.kn), sequence_ptr=ptr(self.sequence), stream=stream)
        self.cache.attend(ptr(self.q), m, QH, ptr(self.lengths), ptr(self.rows), PAGES, ptr(self.attn), BF16,
                          scale=ref.softmax_scale(D), **ws)
        self.out.handle.linear(ptr(self.attn), m, ptr(self.block), F32, **ws)
        ops.norm_device(ptr(self.block), F32, m, H, post_weight_ptr=ptr(self.post), gate_ptr=ptr(self.gate), scale=0.5,
                        residual_ptr=ptr(self.stream), hidden_ptr=ptr(self.after), weight_ptr=ptr(self.pre),
                        y_ptr=ptr(self.y), y_type=BF16, stream=stream)

    def check(self, tokens, what):
        m = len(tokens)
        bits = lambda t: t.cpu().view(torch.int16).numpy().view(np.uint16)  # noqa: E731
        print(f"[gpu] {what}: {m} tokens", flush=True)
        _, want, _, off = ref.norm(self.stream[:m], weight=self.pre)
        close(self.x[:m], want, off, BF16, what + " norm")
        check(self.heads[:m], expected(self.qkv, bits(self.x[:m]), 0, None, None, None, F32), what + " qkv")
        heads = self.heads[:m].view(m, QH + 2 * KV, D)
        angles = BASE ** (-2.0 * np.arange(D // 2) / D)
        for part, weight, got in ((heads[:, :QH], self.qn, self.q[:m]), (heads[:, QH:QH + KV], self.kn, None),
                                  (heads[:, QH + KV:], None, None)):
            at = torch.tensor([p for _, p in tokens])
            numbers = self.table.cpu()[[s for s, _ in tokens], at // PAGE].long()
            if weight is None:
                close(self.v.cpu()[numbers, :, at % PAGE], ref.f64(part), torch.zeros(1, dtype=torch.float64), self.type, what + " v")
                continue
            want, off = ref.head_norm(part, weight, 1e-6)
            want, off = ref.rotate(want, at, angles, 1.0, False, off)
            close(self.k.cpu()[numbers, :, at % PAGE] if got is None else got, want, off, self.type, what + " heads")
        k, v, table = self.k.cpu(), self.v.cpu(), self.table.cpu().numpy()
        for i, (s, p) in enumerate(tokens):
            want, off = ref.attention(self.q[i], ref.gather(k, table[s], p + 1), ref.gather(v, table[s], p + 1),
                                      scale=ref.softmax_scale(D))
            close(self.attn[i].view(QH, D), want, off, BF16, f"{what} attention of {s}, {p}")
        check(self.block[:m], expected(self.out, bits(self.attn[:m]), 0, None, None, None, F32), what + " out")
        eh, ey, h_off, y_off = ref.norm(self.block[:m], post=self.post, gate=self.gate, scale=0.5, residual=self.stream[:m],
                                        weight=self.pre)
        close(self.after[:m], eh, h_off, F32, what + " residual stream")
        close(self.y[:m], ey, y_off, BF16, what + " norm behind")


@pytest.mark.parametrize("kind,cache_type", [(syn.Q8_0, BF16), (syn.Q4_K, _native.F16)])
def test_prompt_then_decoded_tokens(kind, cache_type):
    ops.init(0)
    prompt = [(s, p) for s, n in enumerate(PROMPTS) for p in range(n)]
    layer = Layer(kind, cache_type, len(prompt), 60)
    eager, side = torch.cuda.current_stream().cuda_stream, torch.cuda.Stream()
    layer.inputs(prompt)
    layer.run(len(prompt), eager)
    torch.cuda.synchronize()
    layer.check(prompt, "prompt")
    m = len(PROMPTS)

    def tokens(step):
        return [(s, n + step) for s, n in enumerate(PROMPTS)]

    layer.inputs(tokens(0))
    layer.run(m, eager)
    torch.cuda.synchronize()
    layer.check(tokens(0), "first token")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer.run(m, side.cuda_stream)
    for step in range(1, 6):
        layer.inputs(tokens(step))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t[:m].clone() for t in (layer.x, layer.q, layer.attn, layer.after, layer.y)]
        layer.check(tokens(step), f"replay {step}")
        layer.run(m, eager)  # the same places again: the same values
        torch.cuda.synchronize()
        for a, b in zip(replayed, (layer.x, layer.q, layer.attn, layer.after, layer.y)):
            assert torch.equal(a, b[:m]), step
