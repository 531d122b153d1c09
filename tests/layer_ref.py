"""Norms, rotary positions and attention over a paged cache from their definitions,
in float64 on the CPU, and how far a kernel in fp32 may be from them."""
import math

import numpy as np
import torch

F32, F16, BF16 = 0, 1, 30
DTYPE = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
STEP = 2.0**-24  # half a step of fp32


def half_step(y, type_id):
    """What rounding to the type costs: relative, and in fp16's subnormals absolute."""
    eps = torch.finfo(DTYPE[type_id]).eps / 2
    return eps * y.abs() + (2.0**-25 if type_id == F16 else 0.0)


def f64(t):
    return None if t is None else t.detach().cpu().to(torch.float64)


def unit(v, layer, eps):
    if layer:
        v = v - v.mean(-1, keepdim=True)
    return v / (v.square().mean(-1, keepdim=True) + eps).sqrt()


def norm(x, *, post=None, gate=None, scale=1.0, residual=None, weight=None, bias=None, layer=False, eps=1e-6):
    """hidden, y and how far each may be off before its own rounding.

    A row's sums pass through at most 64 additions of a thread and 22 of the
    workgroup, 86 STEP of the sum of magnitudes: 43 on the root and 86 of the largest
    element on a mean, for each of the two norms; 256 STEP of the row's largest
    magnitude, scaled as the element is, holds all of them and the products."""
    x, post, gate, residual, weight, bias = (f64(t) for t in (x, post, gate, residual, weight, bias))
    b = x if post is None else unit(x, layer, eps) * post
    off = 4 * STEP * b.abs()
    if post is not None:
        r = 1.0 / ((x - x.mean(-1, keepdim=True) if layer else x).square().mean(-1, keepdim=True) + eps).sqrt()
        off = 256 * STEP * x.abs().amax(-1, keepdim=True) * r * post.abs()
    g = scale * (1.0 if gate is None else gate)
    h = b * g
    off = off * (abs(scale) if gate is None else abs(scale) * gate.abs()) + 4 * STEP * h.abs()
    if residual is not None:
        h = h + residual
        off = off + STEP * (h.abs() + residual.abs())
    centred = h - h.mean(-1, keepdim=True) if layer else h
    r = 1.0 / (centred.square().mean(-1, keepdim=True) + eps).sqrt()
    y = centred * r
    y_off = (256 * STEP * h.abs().amax(-1, keepdim=True) + 2 * off.amax(-1, keepdim=True)) * r
    if weight is not None:
        y, y_off = y * weight, y_off * weight.abs()
    if bias is not None:
        y, y_off = y + bias, y_off + STEP * ((y + bias).abs() + bias.abs())
    return h, y, off, y_off


def rotate(x, positions, angles, magnitude, interleaved, off=None):
    """x (tokens, heads, dim), its first 2 len(angles) elements turned, and how far
    off: the angle in revolutions is rounded to fp32 once (2^-25, 2^-22.3 in radians),
    the sine and cosine are 2 steps off, then two products and a sum: 24 STEP of
    |a| + |b|."""
    x = f64(x)
    off = torch.zeros_like(x) if off is None else off
    n = len(angles)
    t = f64(positions)[:, None, None] * torch.as_tensor(np.asarray(angles, np.float64))
    i = torch.arange(n)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    a, b = x[..., first], x[..., second]
    y, far = x.clone(), off.clone()
    c, s = magnitude * t.cos(), magnitude * t.sin()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    both = 24 * STEP * magnitude * (a.abs() + b.abs()) + magnitude * (off[..., first] + off[..., second])
    far[..., first], far[..., second] = both, both
    return y, far


def head_norm(x, weight, eps):
    """RMS norm of heads: 86 STEP as in norm(), and the products."""
    x, w = f64(x), f64(weight)
    y = unit(x, False, eps) * w
    return y, 64 * STEP * y.abs()


def attention(q, k, v, *, scale, softcap=0.0, sinks=None):
    """One sequence: q (heads, dim), k and v (keys, kv_heads, dim) -> out (heads, dim)
    and how far off before its own rounding: E = (dim + 8) STEP scale |q| . |k| on a
    score in any order of addition, 4 STEP of the score (its scaling by log2 e) and
    STEP 16 of a cap; twice that on every weight, 2^-17 for a weight in two parts of 8
    bits, and one STEP a key for the sums, all of sum p |v|."""
    q, k, v, sinks = f64(q), f64(k), f64(v), f64(sinks)
    heads, dim = q.shape
    n, kv_heads = k.shape[:2]
    if n == 0:
        return torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dim, dtype=torch.float64)
    group = heads // kv_heads
    kk, vv = k.transpose(0, 1).repeat_interleave(group, 0), v.transpose(0, 1).repeat_interleave(group, 0)
    s = scale * torch.bmm(kk, q[:, :, None])[:, :, 0]
    near = (dim + 8) * STEP * abs(scale) * torch.bmm(kk.abs(), q.abs()[:, :, None])[:, :, 0] + 4 * STEP * s.abs()
    if softcap:
        s = softcap * torch.tanh(s / softcap)
        near = near + 16 * STEP * softcap
    top = s.amax(1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks[:, None])
    p = torch.exp(s - top)
    total = p.sum(1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks[:, None] - top)
    p = p / total
    out = torch.bmm(p[:, None, :], vv)[:, 0]
    size = torch.bmm(p[:, None, :], vv.abs())[:, 0]
    return out, (2 * near.amax(1, keepdim=True) + 2.0**-17 + (n + 16) * STEP) * size


def gather(cache, table_row, count, begin=0):
    """Tokens begin .. count - 1 of a sequence as (tokens, kv_heads, dim)."""
    pages, kv_heads, page, dim = cache.shape
    at = np.arange(begin, count)
    page_of = torch.as_tensor(np.asarray(table_row)[at // page].astype(np.int64))
    return cache[page_of, :, torch.as_tensor(at % page)]


def softmax_scale(dim):
    return 1.0 / math.sqrt(dim)
