"""Performance cases of what stands between a decoder layer's quantized products.

Four operators take a layer from one product to the next: the norms before and
after a block with its gate, scale and residual; rotary positions; the new keys
and values, normalised and rotated, appended to a paged cache; and the attention
of one new token a sequence over that cache.  Each case is one call at the sizes
of 7B-class and 128-expert models; draw() gives others of the same ranges.

own = False computes the operators in plain torch operations, own = True
through the library's device entry points.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

ELEMENT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ELEMENT_ID = {"f32": 0, "f16": 1, "bf16": 30}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
KIND = {"rms": 0, "layer": 1}
LAYOUT = {"half": 0, "interleaved": 1}
# how positions are scaled: the library's number, then its factor, original context, low and high
SCALING = {"none": (0, 1.0, 0.0, 0.0, 0.0), "linear": (1, 4.0, 0.0, 0.0, 0.0), "yarn": (2, 4.0, 32768.0, 1.0, 32.0),
           "llama3": (3, 8.0, 8192.0, 1.0, 4.0)}
GOLDEN = (math.sqrt(5.0) - 1.0) / 2.0


def listed():
    def norm(name, rows, cols, x="bf16", hidden="bf16", y="bf16", kind="rms", post=False, gate=False, residual=True,
             bias=False, scale=1.0):
        return {"name": name, "op": "norm", "rows": rows, "cols": cols, "x": x, "hidden": hidden, "y": y, "kind": kind,
                "post": post, "gate": gate, "residual": residual, "bias": bias, "scale": scale}

    def rope(name, tokens, heads, dim, rot, type, layout="half", scaling="none", base=10000.0, start=0):
        return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "dim": dim, "rot": rot, "type": type,
                "layout": layout, "scaling": scaling, "base": base, "start": start}

    def append(name, tokens, sequences, q_heads, kv_heads, dim, type, cache, page=16, layout="half", rot=None,
               scaling="none", base=500000.0, normed=False, start=0):
        return {"name": name, "op": "append", "tokens": tokens, "sequences": sequences, "q_heads": q_heads,
                "kv_heads": kv_heads, "dim": dim, "rot": rot or dim, "type": type, "cache": cache, "page": page,
                "layout": layout, "scaling": scaling, "base": base, "normed": normed, "start": start}

    def attend(name, sequences, length, q_heads, kv_heads, dim, cache, out="bf16", page=16, window=0, sinks=False, cap=0.0):
        return {"name": name, "op": "attend", "sequences": sequences, "length": length, "q_heads": q_heads,
                "kv_heads": kv_heads, "dim": dim, "cache": cache, "out": out, "page": page, "window": window,
                "sinks": sinks, "cap": cap}

    return [
        # One decoded token: the residual stream in 32 bits, the next product's input in bf16.
        norm("norm_1x4096", 1, 4096, hidden="f32"),
        # A short prompt at a hidden size that is no multiple of 256, layer norm with its bias.
        norm("norm_100x2880_layer", 100, 2880, x="f16", hidden="f16", y="f16", kind="layer", bias=True),
        # A long prompt's chunk: the norm after a block, its gate and scale, and the next block's norm.
        norm("norm_8192x4096_post", 8192, 4096, post=True, gate=True, scale=0.5),
        # A short prompt, a part of each head rotated, in neighbouring pairs.
        rope("rope_333x32x64", 333, 32, 64, 32, "f32", layout="interleaved"),
        # A chunk of a long prompt, far positions.
        rope("rope_4096x32x128", 4096, 32, 128, 128, "bf16", scaling="yarn", base=1000000.0, start=100000),
        # One decoded token, from a mat-vec's 32-bit result into a cache of f16.
        append("append_1_f32", 1, 1, 32, 8, 128, "f32", "f16", scaling="llama3", start=3001),
        # 64 sequences decoding together, heads normalised before they turn.
        append("append_64_normed", 64, 64, 32, 4, 128, "bf16", "bf16", base=1000000.0, normed=True, start=1000),
        # A prompt's chunk, three sequences in it.
        append("append_4096_prompt", 4096, 3, 32, 8, 128, "bf16", "bf16", scaling="llama3", page=64),
        # One sequence, short: latency.
        attend("attend_1x700", 1, 700, 32, 8, 128, "f16", out="f16"),
        # One sequence of 128k tokens, four heads of keys and values.
        attend("attend_1x131072", 1, 131072, 32, 4, 128, "bf16"),
        # A batch of ragged lengths, the largest call.
        attend("attend_64x8192", 64, 8192, 32, 8, 128, "bf16"),
        # Many sequences through a layer of a sliding window with sinks, heads of 64.
        attend("attend_256_window", 256, 2048, 64, 8, 64, "f16", window=128, sinks=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "norm", "rope", "append", "append", "attend", "attend", "attend"))
    types = ("bf16", "bf16", "f16", "f32")
    if op == "norm":
        cols = 8 * _log_int(rng, 32, 1792) if rng.random() < 0.8 else _log_int(rng, 200, 9000)
        rows = min(_log_int(rng, 1, 8192), 8192 * 4096 // cols)
        post = rng.random() < 0.4
        return {"op": op, "rows": rows, "cols": cols, "x": rng.choice(types), "hidden": rng.choice(types),
                "y": rng.choice(types), "kind": rng.choice(("rms", "rms", "layer")), "post": post,
                "gate": rng.random() < 0.3, "residual": rng.random() < 0.8, "bias": rng.random() < 0.3,
                "scale": rng.choice((1.0, 1.0, 0.22))}
    dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
    turn = {"layout": rng.choice(("half", "half", "interleaved")), "rot": rng.choice((dim, dim, dim // 2, dim // 4)),
            "scaling": rng.choice(("none", "none", "linear", "yarn", "llama3")),
            "base": rng.choice((10000.0, 500000.0, 1000000.0))}
    if op == "rope":
        heads = rng.randint(1, 64)
        tokens = min(_log_int(rng, 1, 4096), 4096 * 32 * 128 // (heads * dim))
        return {"op": op, "tokens": tokens, "heads": heads, "dim": dim, "type": rng.choice(types),
                "start": rng.choice((0, 5000, 100000)), **turn}
    kv_heads = rng.choice((1, 2, 4, 8, 8))
    q_heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    page = rng.choice((16, 16, 32, 64, 128))
    if op == "append":
        tokens = min(_log_int(rng, 1, 4096), 4096 * 48 * 128 // ((q_heads + 2 * kv_heads) * dim))
        sequences = tokens if rng.random() < 0.5 and tokens <= 256 else rng.randint(1, min(tokens, 8))
        return {"op": op, "tokens": tokens, "sequences": sequences, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
                "type": rng.choice(types), "cache": rng.choice(("bf16", "f16")), "page": page,
                "normed": rng.random() < 0.4, "start": rng.choice((0, 37, 1000)), **turn}
    sequences = _log_int(rng, 1, 256)
    most = 40 * 8192 * 8 * 128 // (sequences * kv_heads * dim)
    length = _log_int(rng, 1, max(2, min(131072, most)))
    return {"op": op, "sequences": sequences, "length": length, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "cache": rng.choice(("bf16", "f16")), "out": rng.choice(types), "page": page,
            "window": rng.choice((0, 0, 0, 128, 1000)), "sinks": rng.random() < 0.25,
            "cap": rng.choice((0.0, 0.0, 0.0, 50.0))}


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 29)
    return g


def _normal(g, shape, sigma=1.0, dtype=torch.float32):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, sigma, generator=g)


def _lengths(case):
    """The cached tokens of each sequence: the first has `length`, the others a quarter to all of it."""
    n = case["length"]
    return [n] + [max(1, int(n * (0.25 + 0.75 * ((i * GOLDEN) % 1.0)))) for i in range(1, case["sequences"])]


def _page_table(g, needed, columns):
    """(rows, columns) page numbers in a shuffled pool, `needed` of each row in use; the pool's pages."""
    pool = int(sum(needed)) + 1  # page 0 stands for no page
    order = (torch.randperm(pool - 1, device="cuda", generator=g) + 1).to(torch.int32)
    need = torch.tensor(needed, device="cuda")
    at = torch.arange(columns, device="cuda").unsqueeze(0)
    used = at < need.unsqueeze(1)
    index = (need.cumsum(0) - need).unsqueeze(1) + at
    table = torch.where(used, order[torch.where(used, index, 0)], 0)
    return table.to(torch.int32).contiguous(), pool


def _norm_inputs(case, g):
    shape, cols = (case["rows"], case["cols"]), case["cols"]
    x = _normal(g, shape)
    x[:, ::97] *= 12.0  # a few large channels
    s = {"x": x.to(ELEMENT[case["x"]]), "weight": 1.0 + _normal(g, (cols,), 0.2)}
    s["post"] = 1.0 + _normal(g, (cols,), 0.2) if case["post"] else None
    s["gate"] = _normal(g, (cols,), 0.5) if case["gate"] else None
    s["bias"] = _normal(g, (cols,), 0.2) if case["bias"] else None
    s["residual"] = _normal(g, shape, 3.0).to(ELEMENT[case["hidden"]]) if case["residual"] else None
    return s


def _rope_inputs(case, g):
    n = case["tokens"]
    x = _normal(g, (n, case["heads"], case["dim"])).to(ELEMENT[case["type"]])
    return {"x": x, "positions": (case["start"] + torch.arange(n, device="cuda")).to(torch.int32)}


def _append_inputs(case, g):
    n, count, page = case["tokens"], case["sequences"], case["page"]
    width = (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]
    s = {"qkv": _normal(g, (n, width), 1.5).to(ELEMENT[case["type"]])}  # one product gives all three
    t = torch.arange(n, device="cuda")
    seq = t * count // n
    first = (torch.arange(count, device="cuda") * n + count - 1) // count  # each sequence's first token
    s["sequence"] = seq.to(torch.int32)
    if n == count:  # decoding: each sequence at a place of its own
        s["positions"] = (case["start"] + torch.randint(0, 256, (n,), device="cuda", generator=g)).to(torch.int32)
        last = case["start"] + 255
    else:
        s["positions"] = (case["start"] + t - first[seq]).to(torch.int32)
        last = case["start"] + (n + count - 1) // count - 1
    columns = last // page + 1
    s["table"], pool = _page_table(g, [columns] * count, columns)
    cache = (pool, case["kv_heads"], page, case["dim"])
    s["k"], s["v"] = (_normal(g, cache, 1.0, ELEMENT[case["cache"]]) for _ in range(2))
    s["q_norm"] = 1.0 + _normal(g, (case["dim"],), 0.2) if case["normed"] else None
    s["k_norm"] = 1.0 + _normal(g, (case["dim"],), 0.2) if case["normed"] else None
    return s


def _attend_inputs(case, g):
    lengths, page = _lengths(case), case["page"]
    columns = -(-case["length"] // page)
    mixed = torch.randperm(len(lengths), device="cuda", generator=g)
    at = torch.tensor(lengths, device="cuda")[mixed]
    s = {"lengths": at.to(torch.int32).contiguous()}
    s["table"], pool = _page_table(g, (-(-at // page)).tolist(), columns)
    cache, dtype = (pool, case["kv_heads"], page, case["dim"]), ELEMENT[case["cache"]]
    s["k"], s["v"] = _normal(g, cache, 1.0, dtype), _normal(g, cache, 1.0, dtype)
    # scores of a trained head: a few keys stand out
    s["q"] = _normal(g, (case["sequences"], case["q_heads"], case["dim"]), 2.0).to(dtype)
    s["sinks"] = _normal(g, (case["q_heads"],), 2.0) if case["sinks"] else None
    return s


_INPUTS = {"norm": _norm_inputs, "rope": _rope_inputs, "append": _append_inputs, "attend": _attend_inputs}


def prepare(case, seed):
    s = _INPUTS[case["op"]](case, _gen(seed))
    s["case"] = case
    if case["op"] == "norm":
        s["h"] = torch.zeros((case["rows"], case["cols"]), device="cuda", dtype=ELEMENT[case["hidden"]])
        s["y"] = torch.zeros((case["rows"], case["cols"]), device="cuda", dtype=ELEMENT[case["y"]])
    elif case["op"] == "rope":
        s["out"] = torch.zeros_like(s["x"])
    elif case["op"] == "append":
        s["q_out"] = torch.zeros((case["tokens"], case["q_heads"], case["dim"]), device="cuda", dtype=ELEMENT[case["cache"]])
    else:
        s["out"] = torch.zeros(s["q"].shape, device="cuda", dtype=ELEMENT[case["out"]])
    if case["op"] in ("rope", "append"):
        s["turns"], s["magnitude"] = _frequencies(case)
    if own:
        from gollek_amd import tensor_ops as ops
        ops.init(0)
        s["ops"] = ops
        if case["op"] in ("rope", "append"):
            kind, factor, context, low, high = SCALING[case["scaling"]]
            s["rope"] = ops.Rope(case["rot"], layout=LAYOUT[case["layout"]], base=case["base"], scaling=kind, factor=factor,
                                 original_context=context, low=low, high=high)
        if case["op"] in ("append", "attend"):
            s["cache"] = ops.KvCache(ELEMENT_ID[case["cache"]], s["k"].data_ptr(), s["v"].data_ptr(), s["k"].shape[0],
                                     case["page"], case["kv_heads"], case["dim"])
        need = 0
        if case["op"] == "attend":
            need = s["cache"].attend_workspace_bytes(case["sequences"], case["q_heads"], s["table"].shape[1])
        s["ws"] = torch.zeros(max(need, 256), device="cuda", dtype=torch.uint8)
    return s


# ---- the plain forms --------------------------------------------------------

def _frequencies(case):
    """Radians a position for each pair of a head, in float64, and what cosine and sine are multiplied by."""
    rot, base = case["rot"], case["base"]
    _, factor, context, low, high = SCALING[case["scaling"]]
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    f = torch.exp(i * (-2.0 * math.log(base) / rot))
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":
        def pair(turns):
            return rot * math.log(context / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        first, last = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rot - 1)
        ramp = ((i - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        return f * (1.0 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    if case["scaling"] == "llama3":
        share = ((context * f / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return f * share + f / factor * (1.0 - share), 1.0
    return f, 1.0


def _turned(x, positions, turns, magnitude, rot, layout):
    """x (tokens, heads, dim) float32, its first `rot` elements a head rotated."""
    angle = positions.to(torch.float64).unsqueeze(1) * turns  # 32 bits lose far positions' angles
    c = (torch.cos(angle) * magnitude).to(torch.float32).unsqueeze(1)
    s = (torch.sin(angle) * magnitude).to(torch.float32).unsqueeze(1)
    r = x[:, :, :rot]
    if layout == "half":
        a, b = r[:, :, :rot // 2], r[:, :, rot // 2:]
        r = torch.cat([a * c - b * s, b * c + a * s], 2)
    else:
        a, b = r[:, :, 0::2], r[:, :, 1::2]
        r = torch.stack([a * c - b * s, b * c + a * s], 3).flatten(2)
    return torch.cat([r, x[:, :, rot:]], 2)


def _normed(v, kind, eps=1e-6):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def _plain_norm(s):
    c = s["case"]
    h = s["x"].to(torch.float32)
    if s["post"] is not None:
        h = _normed(h, c["kind"]) * s["post"]
    if s["gate"] is not None:
        h = h * s["gate"]
    h = h * c["scale"]
    if s["residual"] is not None:
        h = h + s["residual"].to(torch.float32)
    y = _normed(h, c["kind"]) * s["weight"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return {"hidden": h.to(ELEMENT[c["hidden"]]), "y": y.to(ELEMENT[c["y"]])}


def _plain_rope(s):
    c = s["case"]
    return _turned(s["x"].to(torch.float32), s["positions"], s["turns"], s["magnitude"], c["rot"],
                   c["layout"]).to(ELEMENT[c["type"]])


def _plain_append(s):
    c = s["case"]
    q, k, v = (t.unflatten(1, (-1, c["dim"])) for t in s["qkv"].split(
        [c["q_heads"] * c["dim"], c["kv_heads"] * c["dim"], c["kv_heads"] * c["dim"]], 1))
    q, k = q.to(torch.float32), k.to(torch.float32)
    if s["q_norm"] is not None:
        q, k = _normed(q, "rms") * s["q_norm"], _normed(k, "rms") * s["k_norm"]
    q = _turned(q, s["positions"], s["turns"], s["magnitude"], c["rot"], c["layout"])
    k = _turned(k, s["positions"], s["turns"], s["magnitude"], c["rot"], c["layout"])
    at = s["positions"].to(torch.int64)
    page = s["table"][s["sequence"].to(torch.int64), at // c["page"]].to(torch.int64).unsqueeze(1)
    head, slot = torch.arange(c["kv_heads"], device=at.device).unsqueeze(0), (at % c["page"]).unsqueeze(1)
    s["k"][page, head, slot] = k.to(s["k"].dtype)
    s["v"][page, head, slot] = v.to(torch.float32).to(s["v"].dtype)
    return {"q": q.to(ELEMENT[c["cache"]]), "k": s["k"], "v": s["v"]}


def _plain_attend(s):
    c = s["case"]
    n, kv, dim = c["sequences"], c["kv_heads"], c["dim"]
    pages = s["table"].to(torch.int64)
    k = s["k"][pages].transpose(1, 2).reshape(n, kv, -1, dim).to(torch.float32)
    v = s["v"][pages].transpose(1, 2).reshape(n, kv, -1, dim).to(torch.float32)
    length = s["lengths"].view(n, 1, 1, 1)
    j = torch.arange(k.shape[2], device=k.device)
    seen = j < length
    if c["window"]:
        seen = seen & (j >= length - c["window"])
    q = s["q"].to(torch.float32).reshape(n, kv, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(dim)
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    score = torch.where(seen, score, -math.inf)
    most = score.max(3, keepdim=True).values
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, kv, -1, 1)
        most = torch.maximum(most, sink)
    p = torch.exp(score - most)
    total = p.sum(3, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - most)
    v = torch.where(seen.transpose(2, 3), v, torch.zeros_like(v))  # what is behind a sequence may be anything
    return (torch.matmul(p, v) / total).reshape(n, -1, dim).to(ELEMENT[c["out"]])


_PLAIN = {"norm": _plain_norm, "rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}


# ---- the library's calls ----------------------------------------------------

def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own_norm(s, stream):
    c = s["case"]
    s["ops"].norm_device(s["x"].data_ptr(), ELEMENT_ID[c["x"]], c["rows"], c["cols"], post_weight_ptr=_ptr(s["post"]),
                         gate_ptr=_ptr(s["gate"]), scale=c["scale"], residual_ptr=_ptr(s["residual"]),
                         hidden_ptr=s["h"].data_ptr(), hidden_type=ELEMENT_ID[c["hidden"]],
                         weight_ptr=s["weight"].data_ptr(), bias_ptr=_ptr(s["bias"]), kind=KIND[c["kind"]], eps=1e-6,
                         y_ptr=s["y"].data_ptr(), y_type=ELEMENT_ID[c["y"]], stream=stream)
    return {"hidden": s["h"], "y": s["y"]}


def _own_rope(s, stream):
    c = s["case"]
    s["rope"].apply_device(s["x"].data_ptr(), ELEMENT_ID[c["type"]], c["tokens"], c["heads"], c["dim"],
                           s["positions"].data_ptr(), s["out"].data_ptr(), stream=stream)
    return s["out"]


def _own_append(s, stream):
    c = s["case"]
    base, dim, size = s["qkv"].data_ptr(), c["dim"], BYTES[c["type"]]
    width = s["qkv"].shape[1]
    s["cache"].append(base + c["q_heads"] * dim * size, base + (c["q_heads"] + c["kv_heads"]) * dim * size,
                      ELEMENT_ID[c["type"]], c["tokens"], s["positions"].data_ptr(), s["table"].data_ptr(), c["sequences"],
                      s["table"].shape[1], rope=s["rope"], k_stride=width, v_stride=width, q_ptr=base,
                      q_heads=c["q_heads"], q_stride=width, q_out_ptr=s["q_out"].data_ptr(), q_norm_ptr=_ptr(s["q_norm"]),
                      k_norm_ptr=_ptr(s["k_norm"]), eps=1e-6, sequence_ptr=s["sequence"].data_ptr(), stream=stream)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_attend(s, stream):
    c = s["case"]
    s["cache"].attend(s["q"].data_ptr(), c["sequences"], c["q_heads"], s["lengths"].data_ptr(), s["table"].data_ptr(),
                      s["table"].shape[1], s["out"].data_ptr(), ELEMENT_ID[c["out"]], scale=1.0 / math.sqrt(c["dim"]),
                      softcap=c["cap"], window=c["window"], sinks_ptr=_ptr(s["sinks"]), ws_ptr=s["ws"].data_ptr(),
                      ws_bytes=s["ws"].numel(), stream=stream)
    return s["out"]


_OWN = {"norm": _own_norm, "rope": _own_rope, "append": _own_append, "attend": _own_attend}


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state, torch.cuda.current_stream().cuda_stream)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    if op == "norm":
        n, cols = case["rows"] * case["cols"], case["cols"]
        each = BYTES[case["x"]] + BYTES[case["hidden"]] * (1 + case["residual"]) + BYTES[case["y"]]
        return {"bytes": n * each + 4 * cols * (1 + case["post"] + case["gate"] + case["bias"]),
                "flops": n * (8.0 + 4.0 * case["post"])}
    if op == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * BYTES[case["type"]] + 4 * case["tokens"], "flops": 3.0 * n}
    if op == "append":
        n = case["tokens"] * (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": n * (BYTES[case["type"]] + 2) + 12 * case["tokens"], "flops": 4.0 * n}
    keys = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
    rows = case["sequences"] * case["q_heads"]
    moved = 2 * keys * case["kv_heads"] * case["dim"] * 2 + rows * case["dim"] * (2 + BYTES[case["out"]])
    return {"bytes": moved + 4 * (keys // case["page"] + case["sequences"]),
            "flops": 4.0 * keys * case["q_heads"] * case["dim"]}


# ---- the definitions in 64 bits ---------------------------------------------

def _exact_turns(case):
    """Each pair's angle a position and the magnitude, pair by pair from the definitions."""
    rot, base = case["rot"], np.float64(case["base"])
    _, factor, context, low, high = SCALING[case["scaling"]]
    angles = np.empty(rot // 2)
    for i in range(rot // 2):
        a = base ** (-2.0 * i / rot)
        if case["scaling"] == "linear":
            a = a / factor
        elif case["scaling"] == "yarn":
            start = math.floor(rot / 2.0 * math.log(context / (2.0 * math.pi * high), case["base"]))
            end = math.ceil(rot / 2.0 * math.log(context / (2.0 * math.pi * low), case["base"]))
            start, end = max(start, 0), min(end, rot - 1)
            part = min(max((i - start) / max(end - start, 0.001), 0.0), 1.0)
            a = a / factor * part + a * (1.0 - part)
        elif case["scaling"] == "llama3":
            wave = 2.0 * math.pi / a
            if wave > context / low:
                a = a / factor
            elif wave > context / high:
                part = (context / wave - low) / (high - low)
                a = (1.0 - part) * a / factor + part * a
        angles[i] = a
    return angles, (1.0 + 0.1 * math.log(factor) if case["scaling"] == "yarn" else 1.0)


def _exact_rotated(case, x, positions):
    """x (tokens, heads, dim) float64: each pair as a complex number times magnitude * exp(i angle)."""
    angles, magnitude = _exact_turns(case)
    rot = case["rot"]
    angle = positions.to(torch.float64)[:, None, None] * torch.from_numpy(angles).to(x.device)
    first = torch.arange(rot // 2, device=x.device) * (1 if case["layout"] == "half" else 2)
    second = first + (rot // 2 if case["layout"] == "half" else 1)
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.full_like(angle, magnitude), angle)
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_unit(v, kind):
    if kind == "layer":
        return (v - v.mean(-1, keepdim=True)) * torch.rsqrt(v.var(-1, unbiased=False, keepdim=True) + 1e-6)
    return v * torch.rsqrt(v.square().sum(-1, keepdim=True) / v.shape[-1] + 1e-6)


def _exact_norm(case, s):
    f64 = {k: None if s[k] is None else s[k].to(torch.float64) for k in ("x", "weight", "post", "gate", "bias", "residual")}
    block = f64["x"]
    if case["post"]:
        block = f64["post"] * _exact_unit(block, case["kind"])
    block = case["scale"] * block
    if case["gate"]:
        block = f64["gate"] * block
    h = block + f64["residual"] if case["residual"] else block
    y = f64["weight"] * _exact_unit(h, case["kind"])
    return {"hidden": h, "y": y + f64["bias"] if case["bias"] else y}


def _exact_rope(case, s):
    return _exact_rotated(case, s["x"].to(torch.float64), s["positions"])


def _exact_append(case, s):
    dim, qn, kn = case["dim"], case["q_heads"], case["kv_heads"]
    all_heads = s["qkv"].to(torch.float64).reshape(case["tokens"], qn + 2 * kn, dim)
    q, k, v = all_heads[:, :qn], all_heads[:, qn:qn + kn], all_heads[:, qn + kn:]
    if case["normed"]:
        q = s["q_norm"].to(torch.float64) * _exact_unit(q, "rms")
        k = s["k_norm"].to(torch.float64) * _exact_unit(k, "rms")
    q, k = _exact_rotated(case, q, s["positions"]), _exact_rotated(case, k, s["positions"])
    kc, vc = s["k"].to(torch.float64), s["v"].to(torch.float64)
    where = s["positions"].cpu().numpy()
    page = s["table"].cpu().numpy()[s["sequence"].cpu().numpy(), where // case["page"]]
    flat = torch.from_numpy(page.astype(np.int64) * case["page"] + where % case["page"]).to(kc.device)
    for cache, new in ((kc, k), (vc, v)):
        rows = cache.transpose(1, 2).reshape(-1, kn, dim)
        rows[flat] = new
        cache.copy_(rows.reshape(cache.shape[0], case["page"], kn, dim).transpose(1, 2))
    return {"q": q, "k": kc, "v": vc}


def _exact_attend(case, s):
    n, kv, dim, page = case["sequences"], case["kv_heads"], case["dim"], case["page"]
    group = case["q_heads"] // kv
    out = torch.empty((n, kv, group, dim), device=s["q"].device, dtype=torch.float64)
    for i, length in enumerate(s["lengths"].tolist()):
        begin = max(0, length - case["window"]) if case["window"] else 0
        used = s["table"][i, begin // page:-(-length // page)].to(torch.int64)
        skip = begin - begin // page * page
        k, v = (s[c][used].to(torch.float64).transpose(0, 1).reshape(kv, -1, dim)[:, skip:skip + length - begin]
                for c in ("k", "v"))
        q = s["q"][i].to(torch.float64).reshape(kv, group, dim)
        for h in range(kv):
            score = q[h] @ k[h].t().contiguous() * dim ** -0.5
            if case["cap"]:
                score = torch.tanh(score / case["cap"]) * case["cap"]
            if case["sinks"]:
                sink = s["sinks"].to(torch.float64).reshape(kv, group)[h].unsqueeze(1)
                weight = torch.softmax(torch.cat([score, sink], 1), 1)[:, :-1]
            else:
                weight = torch.softmax(score, 1)
            out[i, h] = weight @ v[h]
    return out.reshape(n, -1, dim)


_EXACT = {"norm": _exact_norm, "rope": _exact_rope, "append": _exact_append, "attend": _exact_attend}


def exact(case, seed):
    return _EXACT[case["op"]](case, _INPUTS[case["op"]](case, _gen(seed)))
