"""A decoding step's tail as it would run: an attention output projection onto the
residual stream, a gated FFN, the router's product, routed experts, the lm_head and
sampling, eagerly and as one captured graph.  Every stage is checked against float64 on
the inputs that it had."""
import numpy as np
import pytest
import torch

from gollek_amd import _native
from gollek_amd import tensor_ops as ops
from oracle import oracle as o
from tests.test_gpu_linear import Weight, activate, check, expected
from tests.test_gpu_moe_route import compare as compare_routes
from tests.test_gpu_moe_route import reference as route_reference
from tests.test_gpu_sample import compare as compare_tokens

from gollek_amd import synthetic as syn

pytestmark = pytest.mark.gpu

H, I, E, K, V = 512, 768, 16, 4, 5000
ROUTE = dict(n_groups=4, top_groups=2, group_top=2, scale=1.25)
SAMPLE = dict(t=0.9, k=50, p=0.95)


class Step:
    def __init__(self, m, seed):
        self.m = m
        self.out = Weight(syn.Q4_K, H, H, seed)
        self.up = Weight(syn.Q4_K, I, H, seed + 1)
        self.gate = Weight(syn.Q4_K, I, H, seed + 2)
        self.down = Weight(syn.Q6_K, H, I, seed + 3)
        self.router = Weight(syn.Q8_0, E, H, seed + 4)
        self.experts = [Weight(syn.Q4_K, E * I, H, seed + 5), Weight(syn.Q4_K, E * I, H, seed + 6),
                        Weight(syn.Q4_K, E * H, I, seed + 7)]
        self.head = Weight(syn.Q6_K, V, H, seed + 8)
        rng = np.random.default_rng(seed)

        def dev(a, dtype=torch.float32):
            return torch.from_numpy(np.asarray(a, np.float32)).to(dtype).cuda()

        self.attn = torch.zeros((m, H), device="cuda", dtype=torch.bfloat16)
        self.stream_in = torch.zeros((m, H), device="cuda")
        self.out_bias = dev(rng.normal(size=H))
        self.balance = dev(0.05 * rng.normal(size=E))
        z = lambda *s, d=torch.float32: torch.zeros(s, device="cuda", dtype=d)  # noqa: E731
        self.h, self.hb = z(m, H), z(m, H, d=torch.bfloat16)
        self.u, self.f = z(m, I, d=torch.bfloat16), z(m, I, d=torch.bfloat16)
        self.ffn, self.fb = z(m, H), z(m, H, d=torch.bfloat16)
        self.logits = z(m, E)
        self.ids, self.w, self.moe = z(m, K, d=torch.int32), z(m, K), z(m, H)
        self.last = z(m, H, d=torch.bfloat16)
        self.vocab = z(m, V)
        self.uniform = z(m)
        self.tokens, self.probs, self.kept = z(m, d=torch.int32), z(m), z(m, d=torch.int32)
        self.t, self.k, self.p = (torch.full((m,), SAMPLE["t"], device="cuda"),
                                  torch.full((m,), SAMPLE["k"], device="cuda", dtype=torch.int32),
                                  torch.full((m,), SAMPLE["p"], device="cuda"))
        need = [w.handle.linear_workspace_bytes(m) for w in (self.out, self.up, self.gate, self.down, self.router, self.head)]
        need += [ops.moe_workspace_bytes(m, K, H, I, E), ops.sample_workspace_bytes(m, V)]
        self.ws = torch.zeros(max(need), device="cuda", dtype=torch.uint8)

    def linear(self, wt, x, y, stream, **kw):
        kw = {k: (v.data_ptr() if torch.is_tensor(v) else v) for k, v in kw.items()}
        kind = {torch.float32: _native.F32, torch.bfloat16: _native.BF16}[y.dtype]
        wt.handle.linear(x.data_ptr(), self.m, y.data_ptr(), kind, ws_ptr=self.ws.data_ptr(), ws_bytes=self.ws.numel(),
                         stream=stream, **kw)

    def run(self, stream):
        m = self.m
        self.linear(self.out, self.attn, self.h, stream, bias_ptr=self.out_bias, residual_ptr=self.stream_in)
        self.hb.copy_(self.h)
        self.linear(self.up, self.hb, self.u, stream)
        self.linear(self.gate, self.hb, self.f, stream, activation=ops.ACT_SILU, mul_ptr=self.u)
        self.linear(self.down, self.f, self.ffn, stream, residual_ptr=self.h)
        self.ffn.mul_(2.0**-12)  # (random weights make it large)
        self.fb.copy_(self.ffn)
        self.linear(self.router, self.fb, self.logits, stream)
        g, u, d = (w.handle for w in self.experts)
        ops.moe_block_routed_device(g, u, d, E, self.ffn.data_ptr(), self.logits.data_ptr(), _native.F32, m, K,
                                    ops.ROUTER_SIGMOID, self.ids.data_ptr(), self.w.data_ptr(), self.moe.data_ptr(),
                                    self.ws.data_ptr(), self.ws.numel(), bias_ptr=self.balance.data_ptr(), stream=stream,
                                    **ROUTE)
        self.last.copy_(self.moe / self.moe.square().mean(1, keepdim=True).sqrt())
        self.linear(self.head, self.last, self.vocab, stream)
        ops.sample_device(self.vocab.data_ptr(), _native.F32, m, V, self.uniform.data_ptr(), self.tokens.data_ptr(),
                          temperature_ptr=self.t.data_ptr(), top_k_ptr=self.k.data_ptr(), top_p_ptr=self.p.data_ptr(),
                          probs_ptr=self.probs.data_ptr(), kept_ptr=self.kept.data_ptr(), ws_ptr=self.ws.data_ptr(),
                          ws_bytes=self.ws.numel(), stream=stream)

    def inputs(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.attn.copy_(torch.randn(self.m, H, generator=g))
        self.stream_in.copy_(torch.randn(self.m, H, generator=g))
        self.uniform.copy_(torch.rand(self.m, generator=g))
        torch.cuda.synchronize()

    def check(self, what):
        bits = lambda t: t.cpu().view(torch.int16).numpy().view(np.uint16)  # noqa: E731
        f32, bf16 = _native.F32, _native.BF16
        check(self.h, expected(self.out, bits(self.attn), 0, self.out_bias, None, self.stream_in, f32), what + " out")
        check(self.u, expected(self.up, bits(self.hb), 0, None, None, None, bf16), what + " up")
        check(self.f, expected(self.gate, bits(self.hb), ops.ACT_SILU, None, self.u, None, bf16), what + " gate")
        want, tol = expected(self.down, bits(self.f), 0, None, None, self.h, f32)
        check(self.ffn, (want * 2.0**-12, tol * 2.0**-12), what + " down")
        check(self.logits, expected(self.router, bits(self.fb), 0, None, None, None, f32), what + " router")
        ids, w = route_reference(self.logits.double().cpu().numpy(), K, ops.ROUTER_SIGMOID, self.balance.cpu().numpy(),
                                 **ROUTE)
        compare_routes((self.ids.cpu().numpy(), self.w.cpu().numpy()), (ids, w), what + " routes")
        x = self.ffn.double().cpu().numpy()
        gw, uw, dw = (e.w.reshape(E, -1, e.cols) for e in self.experts)
        ref = np.zeros((self.m, H))
        for t in range(self.m):
            for e, wt in zip(ids[t], w[t]):
                ref[t] += wt * (dw[e] @ (activate(ops.ACT_SILU, gw[e] @ x[t]) * (uw[e] @ x[t])))
        assert o.rel_err(self.moe.cpu().numpy().reshape(-1), ref.reshape(-1)) <= 1e-3  # the expert passes' parity bar
        check(self.vocab, expected(self.head, bits(self.last), 0, None, None, None, f32), what + " head")
        compare_tokens([a.cpu().numpy() for a in (self.tokens, self.probs, self.kept)], self.vocab,
                       self.uniform.cpu().numpy(), what + " tokens", **SAMPLE)


@pytest.mark.parametrize("m", [1, 6, 40])
def test_decode_step(m):
    ops.init(0)
    step, side = Step(m, 50 + m), torch.cuda.Stream()
    step.inputs(1)
    step.run(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    step.check("eager")
    with torch.cuda.stream(side):
        step.run(side.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step.run(side.cuda_stream)
    for turn in range(3):
        step.inputs(10 + turn)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (step.h, step.f, step.ffn, step.moe, step.vocab, step.tokens)]
        step.check(f"replay {turn}")
        step.run(torch.cuda.current_stream().cuda_stream)  # eager, between the replays
        torch.cuda.synchronize()
        for a, b in zip(replayed, (step.h, step.f, step.ffn, step.moe, step.vocab, step.tokens)):
            assert torch.equal(a, b), turn


def test_bf16_results_of_the_host_forms_go_on():
    """linear's bf16 logits (uint16 bit patterns) into the host router and sampler."""
    ops.init(0)
    rows, cols, m = 64, 256, 5
    data = syn.matrix(syn.Q8_0, rows, cols, seed=3)
    t = ops.GgufTensor("w", (cols, rows), syn.Q8_0, data.reshape(-1))
    logits = ops.linear(t, syn.activation_bf16(m, cols, seed=4), _native.BF16)
    values = (logits.astype(np.uint32) << 16).view(np.float32)
    for a, b in zip(ops.moe_route(logits, 6, ops.ROUTER_SOFTMAX, n_groups=8, top_groups=4),
                    ops.moe_route(values, 6, ops.ROUTER_SOFTMAX, n_groups=8, top_groups=4)):
        assert np.array_equal(a, b)
    u = np.linspace(0.05, 0.95, m).astype(np.float32)
    for a, b in zip(ops.sample(logits, u, temperature=20.0, top_p=0.9), ops.sample(values, u, temperature=20.0, top_p=0.9)):
        assert np.array_equal(a, b)
    t.close()
