"""The token operators from their formulas, in FP64, for the tests; and the bounds their kernels keep.

u(dtype) is the largest relative error of one rounding to the type.  Every kernel computes in FP32
(unit 2^-24) and rounds once, so each bound is u |result| plus an FP32 term that counts the longest
chain of roundings, against the magnitudes that the chain adds up (not their sum, which can cancel)."""

from __future__ import annotations

import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# Half the spacing of the type's subnormals: the smallest absolute error of a rounding.
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
E32 = 2.0 ** -24


def rotary(x, positions, frequencies, pairs, interleaved):
    """Rotated x in FP64 and the bound of its error."""
    x64 = x.double()
    n = sum(pairs)
    axis = [0] * pairs[0] + [1] * pairs[1] + [2] * pairs[2]
    angle = positions.double()[:, axis] * frequencies.double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    first = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    second = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    out, size = x64.clone(), torch.zeros_like(x64)
    a, b = x64[..., first], x64[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    size[..., first] = size[..., second] = a.abs() + b.abs()
    # angle to FP32 (|angle| <= pi: half an ulp is 2^-23), cosine and sine within 2 ulp, product, sum
    bound = U[x.dtype] * out.abs() + TINY[x.dtype] + 8 * E32 * size
    bound[..., 2 * n:] = 0  # copied
    return out, bound


def normalised(x, kind, eps):
    """N(x) and, for the bounds, the factor that scales an error of x."""
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    return x * r, r


def norm(x, residual=None, gate=None, post_weight=None, post_bias=None, residual_scale=1.0, kind="rms", weight=None, bias=None,
         scale=None, shift=None, group=None, eps=1e-6):
    """(hidden, bound), (out, bound) in FP64.

    A sum over a row is at most 32 additions in a thread and 10 across threads: 42 roundings, on the
    mean and again on the squares (half of that after the root).  With the few products around
    them 64 FP32 units per norm hold; a second norm doubles them and adds its own."""
    dtype = x.dtype
    wide = lambda t: None if t is None else t.double()
    rows = x.shape[0]
    group = group or max(1, rows)
    at = torch.arange(rows, device=x.device) // group
    mod = lambda t: None if t is None else t.double()[at]
    x, residual, gate, scale, shift = wide(x), wide(residual), mod(gate), mod(scale), mod(shift)
    hidden, size = x, x.abs()
    if residual is not None:
        branch = x
        if post_weight is not None:
            n, r = normalised(x, kind, eps)
            w = post_weight.double()
            branch = n * w + (0 if post_bias is None else post_bias.double())
            size = (size + size.mean(1, keepdim=True)) * r * w.abs() + (0 if post_bias is None else post_bias.double().abs())
            size = size + branch.abs()
        if gate is not None:
            branch, size = branch * gate, size * gate.abs()
        hidden = residual_scale * residual + branch
        size = size + abs(residual_scale) * residual.abs()
    units = 64 * E32 * (1 if post_weight is not None else 1 / 16)  # without a norm: three roundings
    hidden_bound = U[dtype] * hidden.abs() + TINY[dtype] + units * size
    n, r = normalised(hidden, kind, eps)
    w = torch.ones_like(hidden[0]) if weight is None else weight.double()
    y = n * w + (0 if bias is None else bias.double())
    spread = (size + size.mean(1, keepdim=True)) * r * w.abs() + n.abs() * w.abs() * (1 + size.mean(1, keepdim=True) * r)
    spread = spread + (0 if bias is None else bias.double().abs())
    if scale is not None:
        y, spread = y * (1 + scale), spread * (1 + scale.abs())
    if shift is not None:
        y, spread = y + shift, spread + shift.abs()
    return (hidden, hidden_bound), (y, U[dtype] * y.abs() + TINY[dtype] + 128 * E32 * spread)


def append(k, v, k_cache, v_cache, table, starts, lengths):
    """Writes keys and values where the table says, token by token (on lists: the plain meaning)."""
    table, starts, lengths = table.tolist(), starts.tolist(), lengths.tolist()
    pages, page = k_cache.shape[:2]
    for b in range(len(lengths)):
        n = starts[b + 1] - starts[b]
        for i in range(n):
            p = lengths[b] - n + i
            if p < 0 or p // page >= len(table[b]) or not 0 <= table[b][p // page] < pages:
                continue
            k_cache[table[b][p // page], p % page] = k[starts[b] + i]
            v_cache[table[b][p // page], p % page] = v[starts[b] + i]


def visible(position, key, window, sinks, frame):
    qf, kf = position // frame, key // frame
    return (kf <= qf) & ((kf > qf - window) | (kf < sinks)) & (position >= 0)


def attention(q, k_cache, v_cache, table, starts, lengths, window, sinks=0, frame=1, scale=None):
    """out in FP64 and the bound of its error, row by row over the visible keys only.

    A score is a sum of head_dim products (at most head_dim FP32 roundings of their magnitudes); a
    weight's relative error is twice the scores' plus the exponential's, plus u for a weight rounded to
    the type before the second product, with an absolute part where that rounding is to a
    subnormal."""
    dtype, d = q.dtype, q.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    page = k_cache.shape[1]
    ratio = q.shape[1] // k_cache.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    starts, lengths = starts.tolist(), lengths.tolist()
    for b, length in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        if hi <= lo or length <= 0:
            continue
        ids = table[b, :-(-length // page)].long()
        k = k_cache[ids].flatten(0, 1)[:length].double().repeat_interleave(ratio, 1)
        v = v_cache[ids].flatten(0, 1)[:length].double().repeat_interleave(ratio, 1)
        position = torch.arange(length - (hi - lo), length, device=q.device)[:, None]
        seen = visible(position, torch.arange(length, device=q.device)[None], window, sinks, frame)
        used = seen.any(0)
        k, v, seen = k[used], v[used], seen[:, used]
        some = seen.any(1)
        if not bool(some.any()):
            continue
        qq = q[lo:hi].double()[some]
        seen = seen[some][None]
        score = torch.einsum("ihd,khd->hik", qq, k) * scale
        size = torch.einsum("ihd,khd->hik", qq.abs(), k.abs().nan_to_num(0, 0, 0)) * abs(scale)
        score = torch.where(seen, score, -math.inf)
        p = torch.softmax(score, -1)
        # hidden places have no part, whatever they hold
        o = torch.einsum("hik,khd->ihd", p, v.nan_to_num(0, 0, 0))
        mag = torch.einsum("hik,khd->ihd", p, v.abs().nan_to_num(0, 0, 0))
        err = 2 * d * E32 * torch.where(seen, size, 0.0).amax(-1) + 16 * E32 + (U[dtype] if dtype != torch.float32 else 0)
        top = v.abs().nan_to_num(0, 0, 0).amax((0, 2))
        small = TINY[dtype] * seen.sum(-1) * top[:, None] if dtype == torch.float16 else torch.zeros_like(err)
        e = mag * err.T[..., None] + small.T[..., None]
        at = torch.arange(lo, hi, device=q.device)[some]
        out[at] = o
        bound[at] = U[dtype] * o.abs() + TINY[dtype] + 1.01 * e
    return out, bound


def check(got, want, bound):
    """got within bound of want everywhere; both finite."""
    off = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all()), "non-finite output"
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert bool((off <= bound).all()), f"off by {off.max().item():.3g}, {worst:.3g} over its bound"
