"""Performance cases of the operators around the quantized products.

Three operators take over what a GGUF runtime does with a product's result:
the linear layer's epilogue (bias, activation, gate, residual, in the type that
the next layer reads), the router of a mixture of experts (logits to expert ids
and weights, with a balancing bias and groups) and sampling (lm_head logits to
one token per sequence).  Each case is one call at the sizes of 7B-class and
128-expert models; draw() gives others of the same ranges.

own = False computes the operators in plain torch operations, own = True
through the library's device entry points.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = {"q4_0": (32, 18), "q8_0": (32, 34), "q4_k": (256, 144), "q5_k": (256, 176), "q6_k": (256, 210)}
TYPE_ID = {"q4_0": 2, "q8_0": 8, "q4_k": 12, "q5_k": 13, "q6_k": 14}
ELEMENT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ELEMENT_ID = {"f32": 0, "f16": 1, "bf16": 30}
ACTIVATION = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
SCORING = {"softmax": 0, "sigmoid": 1}


def listed():
    def linear(name, kind, m, rows, cols, act="none", out="bf16", bias=False, mul=False, residual=False):
        return {"name": name, "op": "linear", "type": kind, "m": m, "rows": rows, "cols": cols, "act": act, "out": out,
                "bias": bias, "mul": mul, "residual": residual}

    def route(name, tokens, experts, top_k, scoring, bias=False, groups=1, top_groups=1, group_top=1, renormalize=True,
              scale=1.0, type="f32"):
        return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "scoring": scoring,
                "bias": bias, "groups": groups, "top_groups": top_groups, "group_top": group_top,
                "renormalize": renormalize, "scale": scale, "type": type}

    def sample(name, batch, vocab, type, how):
        return {"name": name, "op": "sample", "batch": batch, "vocab": vocab, "type": type, "how": how}

    return [
        # One decoded token: a key / value projection of grouped-query
        # attention with its bias, the smallest product.
        linear("linear_q8_0_m1_1024x4096", "q8_0", 1, 1024, 4096, bias=True),
        # One decoded token: the FFN's down projection onto the residual
        # stream, which is kept in 32 bits.
        linear("linear_q4_k_m1_4096x14336", "q4_k", 1, 4096, 14336, out="f32", residual=True),
        # 16 sequences decoding together: the gate projection, whose SiLU
        # multiplies the up projection's result.
        linear("linear_q4_k_m16_14336x4096", "q4_k", 16, 14336, 4096, act="silu", mul=True),
        # A short prompt at a hidden size that is no multiple of 256.
        linear("linear_q8_0_m100_5760x2880", "q8_0", 100, 5760, 2880, act="gelu_tanh", out="f16", bias=True),
        # A prompt of ragged length: down projection of a Q4_K_M file.
        linear("linear_q6_k_m333_4096x14336", "q6_k", 333, 4096, 14336, out="f32", bias=True, residual=True),
        # A long prompt's chunk: the gate projection, the largest call.
        linear("linear_q4_k_m2048_14336x4096", "q4_k", 2048, 14336, 4096, act="silu", mul=True),
        # The router of one decoded token.
        route("route_t1_e128", 1, 128, 8, "softmax"),
        # A short prompt; sigmoid scores, balanced by a bias, of 4 groups of 8.
        route("route_t256_e256_groups", 256, 256, 8, "sigmoid", bias=True, groups=8, top_groups=4, group_top=2, scale=2.5),
        # A long prompt's chunk, router logits in bf16.
        route("route_t8192_e128", 8192, 128, 8, "softmax", type="bf16"),
        # One sequence: the lm_head's logits over a vocabulary of 128k.
        sample("sample_b1_v128256", 1, 128256, "f32", "top"),
        # A batch of sequences, each with settings of its own.
        sample("sample_b64_v128256", 64, 128256, "f32", "mixed"),
        # A smaller vocabulary, logits in bf16 (many equal values), plain
        # sampling at a temperature.
        sample("sample_b16_v32000", 16, 32000, "bf16", "plain"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear", "route", "route", "sample", "sample"))
    if op == "linear":
        kind = rng.choice(("q4_k", "q4_k", "q5_k", "q6_k", "q8_0", "q4_0"))
        cols = 256 * _log_int(rng, 4, 56)
        if kind in ("q8_0", "q4_0") and rng.random() < 0.25:
            cols = 32 * _log_int(rng, 28, 180)
        rows = _log_int(rng, 256, 14336)
        if rng.random() < 0.75:
            rows = rows // 16 * 16
        m = min(_log_int(rng, 1, 2048), 2048 * 14336 * 4096 // (rows * cols))
        act = rng.choice(("none", "none", "relu", "silu", "gelu", "gelu_tanh"))
        return {"op": op, "type": kind, "m": m, "rows": rows, "cols": cols, "act": act,
                "out": rng.choice(("bf16", "bf16", "f16", "f32")), "bias": rng.random() < 0.5,
                "mul": act != "none" and rng.random() < 0.5, "residual": rng.random() < 0.5}
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        size = rng.choice((4, 8, 16, 20, 32, 48))
        top_groups = rng.randint(1, groups)
        return {"op": op, "tokens": _log_int(rng, 1, 8192), "experts": groups * size, "top_k":
                rng.randint(1, min(10, top_groups * size)), "scoring": rng.choice(("softmax", "sigmoid")),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups, "group_top": rng.choice((1, 2)),
                "renormalize": rng.random() < 0.7, "scale": rng.choice((1.0, 2.5)), "type": rng.choice(("f32", "bf16", "f16"))}
    vocab = _log_int(rng, 1000, 262144)
    return {"op": op, "batch": min(_log_int(rng, 1, 256), 64 * 128256 // vocab), "vocab": vocab,
            "type": rng.choice(("f32", "f32", "bf16", "f16")), "how": rng.choice(("top", "mixed", "plain", "masked"))}


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    return g


def _normal(g, shape, sigma=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, sigma, generator=g)


def _uniform(g, shape, lo, hi):
    return torch.empty(shape, device="cuda").uniform_(lo, hi, generator=g)


def _codes(g, shape, sigma, mid, lo, hi):
    """Bell-shaped integer codes around `mid`, as uint8 (two's complement)."""
    v = torch.empty(shape, device="cuda", dtype=torch.float16).normal_(0.0, sigma, generator=g)
    return v.add_(mid).round_().clamp_(lo, hi).to(torch.int16).to(torch.uint8)


def _halves(x):
    return x.to(torch.float16).view(torch.uint8)


def _packed_blocks(kind, nb, g):
    """(nb, block bytes) uint8: codes and scales distributed as a trained matrix's."""
    if kind == "q8_0":
        return torch.cat([_halves(_uniform(g, (nb, 1), 3e-4, 8e-4)), _codes(g, (nb, 32), 40.0, 0.0, -127, 127)], 1)
    if kind == "q4_0":
        q = _codes(g, (nb, 32), 2.7, 8.0, 0, 15)
        return torch.cat([_halves(_uniform(g, (nb, 1), 4e-3, 1.2e-2)), q[:, :16] | (q[:, 16:] << 4)], 1)
    if kind in ("q4_k", "q5_k"):
        top = 15 if kind == "q4_k" else 31
        d = _uniform(g, (nb, 1), 1e-4, 2.4e-4) * (15.0 / top)
        sc = torch.randint(20, 64, (nb, 8), device="cuda", generator=g, dtype=torch.uint8)
        off = torch.randint(-3, 4, (nb, 8), device="cuda", generator=g, dtype=torch.int16)
        mn = (sc.to(torch.int16) + off).clamp_(0, 63).to(torch.uint8)
        q = _codes(g, (nb, 4, 2, 32), top / 5.6, top / 2.0, 0, top)
        parts = [_halves(d), _halves(d * (top / 2.0)), sc[:, :4] | ((sc[:, 4:] >> 4) << 6),
                 mn[:, :4] | ((mn[:, 4:] >> 4) << 6), (sc[:, 4:] & 15) | ((mn[:, 4:] & 15) << 4)]
        if kind == "q5_k":
            bit = torch.arange(8, device="cuda", dtype=torch.uint8).view(1, 8, 1)
            parts.append(((q.reshape(nb, 8, 32) >> 4) << bit).sum(1, dtype=torch.uint8))
            q &= 15
        return torch.cat(parts + [(q[:, :, 0] | (q[:, :, 1] << 4)).reshape(nb, 128)], 1)
    sc = torch.randint(40, 128, (nb, 16), device="cuda", generator=g, dtype=torch.int16)
    sign = torch.randint(0, 2, (nb, 16), device="cuda", generator=g, dtype=torch.int16)
    q = _codes(g, (nb, 2, 4, 32), 10.0, 32.0, 0, 63)
    low, high = q & 15, q >> 4
    ql = torch.stack([low[:, :, 0] | (low[:, :, 2] << 4), low[:, :, 1] | (low[:, :, 3] << 4)], 2)
    qh = high[:, :, 0] | (high[:, :, 1] << 2) | (high[:, :, 2] << 4) | (high[:, :, 3] << 6)
    return torch.cat([ql.reshape(nb, 128), qh.reshape(nb, 64), (sc * (1 - 2 * sign)).to(torch.uint8),
                      _halves(_uniform(g, (nb, 1), 1.5e-5, 4e-5))], 1)


def _linear_inputs(case, g):
    m, rows, cols = case["m"], case["rows"], case["cols"]
    elements, _ = BLOCK[case["type"]]
    dtype = ELEMENT[case["out"]]
    x = _normal(g, (m, cols))
    x[:, ::256] *= 10.0  # a few large channels
    s = {"w": _packed_blocks(case["type"], rows * (cols // elements), g), "x": x.to(torch.bfloat16)}
    s["bias"] = _normal(g, (rows,), 0.5) if case["bias"] else None
    s["mul"] = _normal(g, (m, rows), 2.0).to(dtype) if case["mul"] else None
    s["residual"] = _normal(g, (m, rows), 2.0).to(dtype) if case["residual"] else None
    return s


def _route_inputs(case, g):
    logits = _normal(g, (case["tokens"], case["experts"]), 1.5).to(ELEMENT[case["type"]])
    return {"logits": logits, "bias": _normal(g, (case["experts"],), 0.05) if case["bias"] else None}


def _sample_inputs(case, g):
    b, v, how = case["batch"], case["vocab"], case["how"]
    logits = _normal(g, (b, v), 2.5)
    # the few tokens that fit the context stand out
    at = torch.randint(0, v, (b, 24), device="cuda", generator=g)
    logits.scatter_(1, at, _uniform(g, (b, 24), 8.0, 16.0))
    if how == "masked":  # a grammar allows one token in 50, and none at all in the last row of a batch
        logits[_uniform(g, (b, v), 0.0, 1.0) > 0.02] = -math.inf
        if b > 1:
            logits[-1] = -math.inf
    n = torch.arange(b, device="cuda")

    def mixed(values, dtype):
        return torch.tensor(values, device="cuda", dtype=dtype)[n % len(values)].contiguous()

    s = {"logits": logits.to(ELEMENT[case["type"]]), "u": _uniform(g, (b,), 0.0, 1.0)}
    s["temperature"] = {"top": torch.full((b,), 0.8, device="cuda"), "plain": torch.full((b,), 1.3, device="cuda"),
                        "mixed": mixed([0.7, 1.0, 0.0, 1.3, 0.8], torch.float32),
                        "masked": mixed([1.0, 0.6], torch.float32)}[how]
    s["top_k"] = {"top": mixed([40], torch.int32), "plain": None, "mixed": mixed([0, 40, 200, 1, 1000, 0, 20], torch.int32),
                  "masked": mixed([64, 0], torch.int32)}[how]
    s["top_p"] = {"top": mixed([0.95], torch.float32), "plain": None,
                  "mixed": mixed([0.9, 1.0, 0.95, 0.8], torch.float32), "masked": mixed([0.9], torch.float32)}[how]
    s["min_p"] = mixed([0.0, 0.05, 0.0], torch.float32) if how in ("mixed", "masked") else None
    return s


_INPUTS = {"linear": _linear_inputs, "route": _route_inputs, "sample": _sample_inputs}


def prepare(case, seed):
    s = _INPUTS[case["op"]](case, _gen(seed))
    s["case"] = case
    if case["op"] == "linear":
        s["y"] = torch.zeros((case["m"], case["rows"]), device="cuda", dtype=ELEMENT[case["out"]])
    elif case["op"] == "route":
        s["ids"] = torch.zeros((case["tokens"], case["top_k"]), device="cuda", dtype=torch.int32)
        s["weights"] = torch.zeros((case["tokens"], case["top_k"]), device="cuda")
    else:
        s["tokens"] = torch.zeros(case["batch"], device="cuda", dtype=torch.int32)
        s["probs"] = torch.zeros(case["batch"], device="cuda")
        s["kept"] = torch.zeros(case["batch"], device="cuda", dtype=torch.int32)
    if own:
        from gollek_amd import tensor_ops as ops
        ops.init(0)
        s["ops"] = ops
        need = 0
        if case["op"] == "linear":
            torch.cuda.synchronize()
            s["handle"] = ops.DeviceWeight(TYPE_ID[case["type"]], s["w"].data_ptr(), case["rows"], case["cols"])
            if case["m"] <= 4:  # a decoding program lays its weights out once
                s["handle"].prepare()
            need = s["handle"].linear_workspace_bytes(case["m"])
        elif case["op"] == "sample":
            need = ops.sample_workspace_bytes(case["batch"], case["vocab"])
        s["ws"] = torch.zeros(max(need, 256), device="cuda", dtype=torch.uint8)
    return s


# ---- the plain forms --------------------------------------------------------

def _half(b, at):
    return b[:, at:at + 2].contiguous().view(torch.float16).to(torch.float32)


def _dequantized(kind, b):
    """(nb, block elements) float32 values of packed blocks."""
    nb = b.shape[0]
    if kind == "q8_0":
        return _half(b, 0) * b[:, 2:].contiguous().view(torch.int8).to(torch.float32)
    if kind == "q4_0":
        return _half(b, 0) * (torch.cat([b[:, 2:] & 15, b[:, 2:] >> 4], 1).to(torch.float32) - 8.0)
    if kind in ("q4_k", "q5_k"):
        s = b[:, 4:16]
        sc = torch.cat([s[:, :4] & 63, (s[:, 8:] & 15) | ((s[:, :4] >> 6) << 4)], 1).to(torch.float32)
        mn = torch.cat([s[:, 4:8] & 63, (s[:, 8:] >> 4) | ((s[:, 4:8] >> 6) << 4)], 1).to(torch.float32)
        qs = b[:, 16 if kind == "q4_k" else 48:].reshape(nb, 4, 32)
        q = torch.stack([qs & 15, qs >> 4], 2).reshape(nb, 8, 32)
        if kind == "q5_k":
            bit = torch.arange(8, device=b.device, dtype=torch.uint8).view(1, 8, 1)
            q = q | (((b[:, None, 16:48] >> bit) & 1) << 4)
        return ((_half(b, 0) * sc).unsqueeze(2) * q.to(torch.float32) - (_half(b, 2) * mn).unsqueeze(2)).reshape(nb, 256)
    ql, qh = b[:, :128].reshape(nb, 2, 2, 32), b[:, 128:192].reshape(nb, 2, 32)
    q = torch.stack([ql[:, :, 0] & 15 | (qh & 3) << 4, ql[:, :, 1] & 15 | (qh >> 2 & 3) << 4,
                     ql[:, :, 0] >> 4 | (qh >> 4 & 3) << 4, ql[:, :, 1] >> 4 | (qh >> 6) << 4], 2).reshape(nb, 16, 16)
    sc = b[:, 192:208].contiguous().view(torch.int8).to(torch.float32)
    return ((_half(b, 208) * sc).unsqueeze(2) * (q.to(torch.float32) - 32.0)).reshape(nb, 256)


def _activated(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_linear(s):
    c = s["case"]
    w = _dequantized(c["type"], s["w"]).reshape(c["rows"], c["cols"])
    y = s["x"].to(torch.float32) @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    y = _activated(y, c["act"])
    if s["mul"] is not None:
        y = y * s["mul"].to(torch.float32)
    if s["residual"] is not None:
        y = y + s["residual"].to(torch.float32)
    return y.to(ELEMENT[c["out"]])


def _plain_route(s):
    c = s["case"]
    l = s["logits"].to(torch.float64)  # two scores may be next to each other
    n, e = l.shape
    if c["scoring"] == "softmax":
        p = torch.exp(l - l.max(1, keepdim=True).values)
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-l))
    choice = p if s["bias"] is None else p + s["bias"].to(torch.float64)
    if c["top_groups"] < c["groups"]:
        grouped = choice.reshape(n, c["groups"], -1)
        best = grouped.sort(dim=2, descending=True).values[:, :, :c["group_top"]].sum(2)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        allowed = torch.zeros((n, c["groups"]), device=l.device, dtype=torch.bool).scatter_(1, order, True)
        choice = torch.where(allowed.unsqueeze(2), grouped, -math.inf).reshape(n, e)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
    w = p.gather(1, ids)
    if c["renormalize"]:
        w = w / w.sum(1, keepdim=True)
    return {"ids": ids.to(torch.int32), "weights": (w * c["scale"]).to(torch.float32)}


def _plain_sample(s):
    l = s["logits"].to(torch.float64)  # sums over a vocabulary, compared with a border
    b, v = l.shape
    top, order = l.sort(dim=1, descending=True, stable=True)
    t = s["temperature"].to(torch.float64).unsqueeze(1)
    greedy = t <= 0
    w = torch.exp((top - top[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    keep = top > -math.inf
    w = torch.where(keep, w, torch.zeros_like(w))
    rank = torch.arange(v, device=l.device).unsqueeze(0)
    if s["top_k"] is not None:
        k = s["top_k"].unsqueeze(1)
        keep = keep & ((k <= 0) | (rank < k))
        w = torch.where(keep, w, torch.zeros_like(w))
    if s["top_p"] is not None:
        p = s["top_p"].to(torch.float64).unsqueeze(1)
        mass = w.cumsum(1)
        keep = keep & ((p >= 1) | (rank == 0) | (mass - w < p * mass[:, -1:]))
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"].to(torch.float64).unsqueeze(1))
    keep = keep & (~greedy | (rank == 0))
    w = torch.where(keep, w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, order, w)  # back to the vocabulary's order
    mass = w.cumsum(1)
    total = mass[:, -1:]
    token = (mass <= s["u"].to(torch.float64).unsqueeze(1) * total).sum(1, keepdim=True).clamp(max=v - 1)
    none = total <= 0
    prob = w.gather(1, token) / torch.where(none, torch.ones_like(total), total)
    return {"tokens": torch.where(none, -1, token)[:, 0].to(torch.int32), "probs": prob[:, 0].to(torch.float32),
            "kept": keep.sum(1).to(torch.int32)}


_PLAIN = {"linear": _plain_linear, "route": _plain_route, "sample": _plain_sample}


# ---- the library's calls ----------------------------------------------------

def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own_linear(s, stream):
    c = s["case"]
    s["handle"].linear(s["x"].data_ptr(), c["m"], s["y"].data_ptr(), ELEMENT_ID[c["out"]], bias_ptr=_ptr(s["bias"]),
                       activation=ACTIVATION[c["act"]], mul_ptr=_ptr(s["mul"]), residual_ptr=_ptr(s["residual"]),
                       ws_ptr=s["ws"].data_ptr(), ws_bytes=s["ws"].numel(), stream=stream)
    return s["y"]


def _own_route(s, stream):
    c = s["case"]
    s["ops"].moe_route_device(s["logits"].data_ptr(), ELEMENT_ID[c["type"]], c["tokens"], c["experts"], c["top_k"],
                              SCORING[c["scoring"]], s["ids"].data_ptr(), s["weights"].data_ptr(), bias_ptr=_ptr(s["bias"]),
                              n_groups=c["groups"], top_groups=c["top_groups"], group_top=c["group_top"],
                              renormalize=c["renormalize"], scale=c["scale"], stream=stream)
    return {"ids": s["ids"], "weights": s["weights"]}


def _own_sample(s, stream):
    c = s["case"]
    s["ops"].sample_device(s["logits"].data_ptr(), ELEMENT_ID[c["type"]], c["batch"], c["vocab"], s["u"].data_ptr(),
                           s["tokens"].data_ptr(), temperature_ptr=_ptr(s["temperature"]), top_k_ptr=_ptr(s["top_k"]),
                           top_p_ptr=_ptr(s["top_p"]), min_p_ptr=_ptr(s["min_p"]), probs_ptr=s["probs"].data_ptr(),
                           kept_ptr=s["kept"].data_ptr(), ws_ptr=s["ws"].data_ptr(), ws_bytes=s["ws"].numel(),
                           stream=stream)
    return {"tokens": s["tokens"], "probs": s["probs"], "kept": s["kept"]}


_OWN = {"linear": _own_linear, "route": _own_route, "sample": _own_sample}


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state, torch.cuda.current_stream().cuda_stream)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    if case["op"] == "linear":
        m, rows, cols = case["m"], case["rows"], case["cols"]
        elements, size = BLOCK[case["type"]]
        out = 4 if case["out"] == "f32" else 2
        moved = rows * cols * size / elements + 2 * m * cols + out * m * rows * (1 + case["mul"] + case["residual"])
        return {"bytes": moved + 4 * rows * case["bias"], "flops": 2.0 * m * rows * cols}
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "route":
        n, e = case["tokens"], case["experts"]
        return {"bytes": n * (e * size + 8 * case["top_k"]) + 4 * e * case["bias"], "flops": 4.0 * n * e}
    return {"bytes": case["batch"] * (case["vocab"] * size + 32), "flops": 4.0 * case["batch"] * case["vocab"]}


# ---- the definitions in 64 bits ---------------------------------------------

def _element_table(kind):
    """For each element of a block: the byte and shift of its low bits, of its high bits, and its scale's number."""
    e = np.arange(BLOCK[kind][0])
    if kind == "q4_0":
        return 2 + e % 16, 4 * (e // 16), None, None, e * 0
    if kind in ("q4_k", "q5_k"):
        at = (48 if kind == "q5_k" else 16) + 32 * (e // 64) + e % 32
        return at, 4 * (e // 32 % 2), 16 + e % 32, e // 32, e // 32
    j, l = e % 128 // 32, e % 32
    return 64 * (e // 128) + 32 * (j % 2) + l, 4 * (j // 2), 128 + 32 * (e // 128) + l, 2 * j, e // 16


def _decoded(kind, b):
    """(nb, block elements) float64, element by element from the formats' layout."""
    def index(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(b.device)

    def half(at):
        return (b[:, at].to(torch.int32) + 256 * b[:, at + 1].to(torch.int32)).to(torch.int16).view(torch.float16).to(torch.float64)

    def signed(v):
        v = v.to(torch.float64)
        return torch.where(v > 127, v - 256, v)

    if kind == "q8_0":
        return signed(b[:, 2:34]) * half(0)[:, None]
    at, shift, high, high_shift, which = _element_table(kind)
    code = (b[:, index(at)].to(torch.int32) >> index(shift)) & 15
    if kind in ("q5_k", "q6_k"):
        bits = 1 if kind == "q5_k" else 3
        code = code + 16 * ((b[:, index(high)].to(torch.int32) >> index(high_shift)) & bits)
    code = code.to(torch.float64)
    if kind == "q4_0":
        return (code - 8.0) * half(0)[:, None]
    if kind == "q6_k":
        return (code - 32.0) * signed(b[:, 192:208])[:, index(which)] * half(208)[:, None]
    s = b[:, 4:16].to(torch.int32)
    scale = [s[:, j] % 64 for j in range(4)] + [s[:, 8 + j] % 16 + 16 * (s[:, j] // 64) for j in range(4)]
    least = [s[:, 4 + j] % 64 for j in range(4)] + [s[:, 8 + j] // 16 + 16 * (s[:, 4 + j] // 64) for j in range(4)]
    scale, least = torch.stack(scale, 1).to(torch.float64), torch.stack(least, 1).to(torch.float64)
    return code * (scale * half(0)[:, None])[:, index(which)] - (least * half(2)[:, None])[:, index(which)]


def _exact_linear(case, s):
    rows, cols, x = case["rows"], case["cols"], s["x"].to(torch.float64)
    per = cols // BLOCK[case["type"]][0]
    step = max(1, (1 << 25) // cols)
    y = torch.cat([x @ _decoded(case["type"], s["w"][r * per:(r + step) * per]).reshape(-1, cols).t().contiguous()
                   for r in range(0, rows, step)], 1)
    if case["bias"]:
        y = y + s["bias"].to(torch.float64)
    if case["act"] == "relu":
        y = y.clamp(min=0.0)
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["act"] == "gelu":
        y = y * torch.special.ndtr(y)
    elif case["act"] == "gelu_tanh":
        y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
    if case["mul"]:
        y = y * s["mul"].to(torch.float64)
    if case["residual"]:
        y = y + s["residual"].to(torch.float64)
    return y


def _exact_route(case, s):
    l = s["logits"].to(torch.float64).cpu().numpy()
    n, e = l.shape
    if case["scoring"] == "softmax":
        p = np.exp(l - np.logaddexp.reduce(l, axis=1)[:, None])
    else:
        p = 0.5 * (1.0 + np.tanh(0.5 * l))
    choice = p + (s["bias"].to(torch.float64).cpu().numpy() if case["bias"] else 0.0)
    groups, size = case["groups"], e // case["groups"]
    best = np.sort(choice.reshape(n, groups, size), 2)[:, :, size - min(size, case["group_top"]):].sum(2)
    place = np.argsort(np.argsort(-best, 1, kind="stable"), 1)  # each group's place
    choice = np.where(np.repeat(place < case["top_groups"], size, 1), choice, -np.inf)
    ids = np.argsort(-choice, 1, kind="stable")[:, :case["top_k"]]
    w = np.take_along_axis(p, ids, 1)
    if case["renormalize"]:
        w = w / w.sum(1, keepdims=True)
    return {"ids": None, "weights": torch.from_numpy(w * case["scale"])}


def _exact_sample(case, s):
    probs = np.zeros(case["batch"])
    host = {k: (None if s[k] is None else s[k].to(torch.float64).cpu().numpy())
            for k in ("logits", "u", "temperature", "top_k", "top_p", "min_p")}
    for b in range(case["batch"]):
        l, t = host["logits"][b], host["temperature"][b]
        at = np.flatnonzero(l > -np.inf)
        if not at.size:
            continue
        at = at[np.lexsort((at, -l[at]))]  # by value, equal ones by index
        if t <= 0:
            probs[b] = 1.0
            continue
        if host["top_k"] is not None and host["top_k"][b] > 0:
            at = at[:int(host["top_k"][b])]
        w = np.exp((l[at] - l[at[0]]) / t)
        if host["top_p"] is not None and host["top_p"][b] < 1:
            n = int(np.searchsorted(np.cumsum(w), host["top_p"][b] * w.sum())) + 1
            at, w = at[:n], w[:n]
        if host["min_p"] is not None:
            at, w = at[w >= host["min_p"][b]], w[w >= host["min_p"][b]]
        w = w[np.argsort(at)]
        chosen = int(np.searchsorted(np.cumsum(w), host["u"][b] * w.sum(), side="right"))
        probs[b] = w[min(chosen, w.size - 1)] / w.sum()
    return {"kept": None, "probs": torch.from_numpy(probs), "tokens": None}


_EXACT = {"linear": _exact_linear, "route": _exact_route, "sample": _exact_sample}


def exact(case, seed):
    return _EXACT[case["op"]](case, _INPUTS[case["op"]](case, _gen(seed)))
