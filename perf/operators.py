"""The token operators' measured cases: their sizes, inputs, plain forms and 64-bit definitions.

The operators restore video streams frame by frame: a tile's features (64x64 positions, as the
deformable convolution leaves them) are cut into tokens, and a block attends from a new frame's
tokens to the frames that a stream keeps in a paged cache.

* rotary     -- rotates heads by their token's (time, row, column) position
* append     -- rotates a step's queries and keys, and writes its keys and values into the cache's pages
* attention  -- attends over the cache: the last `window` frames and the first `sinks` frames are visible
* norm       -- normalises before and after a block, with the block's gate, residual scale and modulation

`run` computes them in their plain form (elementary torch operations in 32 bits, rounded once at the
end) where `own` is false, and through the package where it is true.
"""

import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# --------------------------------------------------------------------------------------- cases


def listed():
    return [
        # One new token of each of four young streams: the call's latency.
        dict(name="attention_token_short", op="attention", dtype="bf16", streams=4, q_lo=1, q_hi=1, kv_lo=1, kv_hi=400,
             q_heads=16, kv_heads=4, head_dim=128, page=16, frame=1, window=256, sinks=4),
        # Decoding token by token for 64 streams whose caches outgrew their window.
        dict(name="attention_token_streams", op="attention", dtype="bf16", streams=64, q_lo=1, q_hi=1, kv_lo=2000,
             kv_hi=12000, q_heads=32, kv_heads=8, head_dim=128, page=64, frame=1, window=4096, sinks=64),
        # One frame (256 tokens: a 64x64 tile in 4x4 patches) of each of eight tile streams, one to 30 frames old.
        dict(name="attention_frame_streams", op="attention", dtype="f16", streams=8, q_lo=256, q_hi=256, kv_lo=256,
             kv_hi=7680, q_heads=16, kv_heads=16, head_dim=64, page=256, frame=256, window=8, sinks=1),
        # Whole 30-frame windows of four tiles at once: the largest products.
        dict(name="attention_clip", op="attention", dtype="f16", streams=4, q_lo=7680, q_hi=7680, kv_lo=7680, kv_hi=7680,
             q_heads=16, kv_heads=8, head_dim=128, page=128, frame=256, window=8, sinks=1),
        # Streams that catch up by unequal steps, seven tokens a frame, three query heads to a key head, pages
        # that end inside a tile.
        dict(name="attention_ragged", op="attention", dtype="bf16", streams=5, q_lo=1, q_hi=61, kv_lo=100, kv_hi=2999,
             q_heads=12, kv_heads=4, head_dim=128, page=48, frame=7, window=100, sinks=2),
        # The queries of one frame.
        dict(name="rotary_frame", op="rotary", dtype="f16", tokens=256, heads=16, head_dim=64, pairs_t=8, pairs_y=12,
             pairs_x=12, interleaved=True),
        # The queries of four 30-frame windows; a few pairs are left as they are.
        dict(name="rotary_clip", op="rotary", dtype="bf16", tokens=30720, heads=16, head_dim=128, pairs_t=16, pairs_y=22,
             pairs_x=22, interleaved=False),
        # One new token of each of eight streams.
        dict(name="append_token", op="append", dtype="bf16", streams=8, q_lo=1, q_hi=1, kv_lo=1, kv_hi=900, q_heads=16,
             kv_heads=4, head_dim=128, page=16, pairs_t=16, pairs_y=24, pairs_x=24, interleaved=False),
        # One to five frames of each of 32 streams.
        dict(name="append_frames", op="append", dtype="f16", streams=32, q_lo=256, q_hi=1280, kv_lo=1280, kv_hi=2048,
             q_heads=16, kv_heads=8, head_dim=128, page=128, pairs_t=16, pairs_y=24, pairs_x=24, interleaved=True),
        # The norm before a block, for one new token of each of eight streams.
        dict(name="norm_token", op="norm", dtype="bf16", rows=8, width=1024, group=1, kind="rms", residual=False,
             post=False, modulated=False, residual_scale=1.0),
        # A block's end and the next one's start for eight 30-frame windows, modulated frame by frame.
        dict(name="norm_clip", op="norm", dtype="f16", rows=61440, width=1024, group=256, kind="layer", residual=True,
             post=False, modulated=True, residual_scale=1.0),
        # An odd width in 32 bits, normalised on both sides of the block.
        dict(name="norm_odd", op="norm", dtype="f32", rows=1003, width=1155, group=59, kind="rms", residual=True, post=True,
             modulated=True, residual_scale=0.875),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))) - 0.5)))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "append", "norm"])
    if op == "rotary":
        head_dim = rng.choice([64, 128, 2 * rng.randint(20, 64)])
        t = rng.randint(0, head_dim // 6)
        y, x = rng.randint(1, head_dim // 6), rng.randint(1, head_dim // 6)
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), tokens=_spread(rng, 1, 15000), heads=_spread(rng, 1, 16),
                    head_dim=head_dim, pairs_t=t, pairs_y=y, pairs_x=x, interleaved=rng.random() < 0.5)
    if op == "norm":
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), rows=_spread(rng, 1, 30000), width=_spread(rng, 64, 2040),
                    group=_spread(rng, 1, 300), kind=rng.choice(["rms", "layer"]), residual=rng.random() < 0.7,
                    post=rng.random() < 0.4, modulated=rng.random() < 0.7, residual_scale=rng.choice([1.0, 0.875, 1.25]))
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    q_heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
    head_dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    dtype = rng.choice(["f16", "bf16"])
    streams = _spread(rng, 1, 24)
    if op == "append":
        q_hi = _spread(rng, 1, 1200)
        kv_hi = q_hi + _spread(rng, 1, 800)
        pairs = head_dim // 2
        t = rng.randint(1, pairs // 2)
        y = rng.randint(0, (pairs - t) // 2)
        return dict(op=op, dtype=dtype, streams=streams, q_lo=rng.randint(1, q_hi), q_hi=q_hi, kv_lo=q_hi, kv_hi=kv_hi,
                    q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, pairs_t=t, pairs_y=y,
                    pairs_x=pairs - t - y, interleaved=rng.random() < 0.5)
    q_hi = rng.choice([1, 1, _spread(rng, 2, 2000)])
    kv_hi = q_hi + _spread(rng, 1, 6000)
    frame = rng.choice([1, 1, rng.randint(2, 300)])
    # A long step of many streams is cut down to what the largest listed case costs.
    while streams > 1 and (streams * q_hi * kv_hi * q_heads * head_dim > 2e10 or streams * kv_hi * kv_heads * head_dim > 2e8):
        streams -= 1
    return dict(op=op, dtype=dtype, streams=streams, q_lo=rng.randint(1, q_hi), q_hi=q_hi, kv_lo=q_hi + rng.randint(0, kv_hi - q_hi),
                kv_hi=kv_hi, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, frame=frame,
                window=_spread(rng, 1, max(2, kv_hi // frame)), sinks=rng.choice([0, 1, rng.randint(0, 8)]))


def _between(lo, hi, n):
    """n lengths from lo to hi in equal steps."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _lengths(case):
    q = _between(case["q_lo"], case["q_hi"], case["streams"])
    kv = _between(case["kv_lo"], case["kv_hi"], case["streams"])
    return q, [max(a, b) for a, b in zip(q, kv)]


# --------------------------------------------------------------------------------------- inputs


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _positions(gen, tokens):
    """(time, row, column) of each token: frames of a stream up to a minute old, 16x16 patches."""
    t = torch.randint(0, 1800, (tokens, 1), generator=gen, device="cuda")
    yx = torch.randint(0, 16, (tokens, 2), generator=gen, device="cuda")
    return torch.cat([t, yx], 1).to(torch.int32)


def _frequencies(case):
    """Radians a position step of each pair, each axis with its own series."""
    series = []
    for n in (case["pairs_t"], case["pairs_y"], case["pairs_x"]):
        series += [10000.0 ** (-i / n) for i in range(n)]
    return torch.tensor(series, dtype=torch.float64, device="cuda")


def _paged(case, gen, dtype):
    """A cache of shuffled pages, all of it holding values, and the streams' places in it."""
    q, kv = _lengths(case)
    page = case["page"]
    need = [-(-n // page) for n in kv]
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(kv), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (total, page, case["kv_heads"], case["head_dim"])
    starts = torch.tensor(np.concatenate([[0], np.cumsum(q)]), dtype=torch.int32, device="cuda")
    return dict(k_cache=_normal(gen, shape, dtype), v_cache=_normal(gen, shape, dtype), table=table, starts=starts,
                lengths=torch.tensor(kv, dtype=torch.int32, device="cuda"), max_q=max(q), max_kv=max(kv), tokens=sum(q))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "rotary":
        s["x"] = _normal(gen, (case["tokens"], case["heads"], case["head_dim"]), dtype)
        s["positions"] = _positions(gen, case["tokens"])
        s["frequencies"] = _frequencies(case)
    elif case["op"] == "append":
        s |= _paged(case, gen, dtype)
        # One projection's output holds a token's queries, keys and values side by side.
        heads = case["q_heads"] + 2 * case["kv_heads"]
        s["qkv"] = _normal(gen, (s["tokens"], heads, case["head_dim"]), dtype)
        s["positions"] = _positions(gen, s["tokens"])
        s["frequencies"] = _frequencies(case)
    elif case["op"] == "attention":
        s |= _paged(case, gen, dtype)
        s["q"] = _normal(gen, (s["tokens"], case["q_heads"], case["head_dim"]), dtype, 1.5)
    else:
        rows, width = case["rows"], case["width"]
        groups = -(-rows // case["group"])
        s["x"] = _normal(gen, (rows, width), dtype, 2.0) + 0.25
        s["weight"] = 1 + _normal(gen, (width,), dtype, 0.1)
        s["bias"] = _normal(gen, (width,), dtype, 0.1) if case["kind"] == "layer" else None
        s["residual"] = _normal(gen, (rows, width), dtype, 3.0) if case["residual"] else None
        s["post_weight"] = 1 + _normal(gen, (width,), dtype, 0.1) if case["residual"] and case["post"] else None
        # One projection of a group's conditioning holds its shift, scale and gate side by side.
        s["modulation"] = _normal(gen, (groups, 3, width), dtype, 0.3) if case["modulated"] else None
    return s


# --------------------------------------------------------------------------------------- plain forms


def _rotate(x, positions, frequencies, case):
    """x [tokens, heads, head_dim] in 32 bits, rotated."""
    counts = [case["pairs_t"], case["pairs_y"], case["pairs_x"]]
    pairs = sum(counts)
    axis = torch.repeat_interleave(torch.arange(3, device=x.device), torch.tensor(counts, device=x.device), output_size=pairs)
    angle = positions[:, axis].float() * frequencies.float()
    c, s = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]
    if case["interleaved"]:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, x[..., 2 * pairs:]], -1)


def _plain_rotary(s):
    return _rotate(s["x"].float(), s["positions"], s["frequencies"], s["case"]).to(s["x"].dtype)


def _places(s):
    """Each token's stream and its position in that stream."""
    starts = s["starts"].long()
    token = torch.arange(s["tokens"], device=starts.device)
    stream = torch.searchsorted(starts[1:], token, right=True)
    return stream, s["lengths"].long()[stream] - starts[stream + 1] + token


def _plain_append(s):
    case = s["case"]
    hq, hk = case["q_heads"], case["kv_heads"]
    stream, position = _places(s)
    page = s["table"][stream, position // case["page"]].long()
    turned = _rotate(s["qkv"][:, :hq + hk].float(), s["positions"], s["frequencies"], case).to(s["qkv"].dtype)
    s["k_cache"][page, position % case["page"]] = turned[:, hq:]
    s["v_cache"][page, position % case["page"]] = s["qkv"][:, hq + hk:]
    return {"q": turned[:, :hq].contiguous(), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _visible(position, key, length, case):
    """Whether the key at `key` is visible to the query at `position` of a stream of `length` tokens."""
    qf, kf = position // case["frame"], key // case["frame"]
    return (kf <= qf) & (key < length) & ((kf > qf - case["window"]) | (kf < case["sinks"])) & (position >= 0)


def _plain_attention(s):
    case = s["case"]
    b, hq, hk, d = case["streams"], case["q_heads"], case["kv_heads"], case["head_dim"]
    table = s["table"].long().clamp(min=0)
    keys = s["k_cache"][table].float().flatten(1, 2).permute(0, 2, 3, 1)  # [streams, kv_heads, head_dim, keys]
    values = s["v_cache"][table].float().flatten(1, 2).permute(0, 2, 1, 3)
    starts, lengths = s["starts"].long(), s["lengths"].long()[:, None]
    steps = starts[1:, None] - starts[:-1, None]
    i = torch.arange(s["max_q"], device=table.device)
    rows = (starts[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[rows].view(b, s["max_q"], hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    position = torch.where(i < steps, lengths - steps + i, -1)[:, :, None]
    key = torch.arange(keys.shape[-1], device=table.device)
    seen = _visible(position, key, lengths[..., None], case)[:, None, None]
    scores = (q @ keys).view(b, hk, hq // hk, s["max_q"], -1) / math.sqrt(d)
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(b, hk, -1, p.shape[-1]) @ values).view(b, hk, hq // hk, s["max_q"], d) / total.clamp(min=1e-37)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, s["max_q"], hq, d)
    return out[i < steps].to(s["q"].dtype)


def _normalised(x, kind, weight, bias, eps=1e-6):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    x = x * weight
    return x if bias is None else x + bias


def _plain_norm(s):
    case = s["case"]
    dtype = s["x"].dtype
    wide = lambda t: None if t is None else t.float()
    x, weight, bias = wide(s["x"]), wide(s["weight"]), wide(s["bias"])
    m = None
    if s["modulation"] is not None:
        m = wide(s["modulation"])[torch.arange(case["rows"], device=x.device) // case["group"]]
    hidden = x
    if s["residual"] is not None:
        if s["post_weight"] is not None:
            x = _normalised(x, case["kind"], wide(s["post_weight"]), None)
        if m is not None:
            x = x * m[:, 2]
        hidden = wide(s["residual"]) * case["residual_scale"] + x
    y = _normalised(hidden, case["kind"], weight, bias)
    if m is not None:
        y = y * (1 + m[:, 1]) + m[:, 0]
    y = y.to(dtype)
    return {"y": y} if s["residual"] is None else {"hidden": hidden.to(dtype), "y": y}


PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention, "norm": _plain_norm}


# --------------------------------------------------------------------------------------- the package


@functools.lru_cache(maxsize=None)
def _ops():
    from jasnamacos_b200.token_ops import CudaTokenOps

    return CudaTokenOps()


def _own(s):
    case, ops = s["case"], _ops()
    if case["op"] == "rotary":
        return ops.rotary(s["x"], s["positions"], s["frequencies"], (case["pairs_t"], case["pairs_y"], case["pairs_x"]),
                          interleaved=case["interleaved"])
    if case["op"] == "append":
        hq, hk = case["q_heads"], case["kv_heads"]
        q, k, v = s["qkv"].split((hq, hk, hk), 1)
        turned = ops.append(k, v, s["k_cache"], s["v_cache"], s["table"], s["starts"], s["lengths"], q=q,
                            positions=s["positions"], frequencies=s["frequencies"],
                            pairs=(case["pairs_t"], case["pairs_y"], case["pairs_x"]), interleaved=case["interleaved"])
        return {"q": turned, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "attention":
        return ops.attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["lengths"], max_q=s["max_q"],
                             max_kv=s["max_kv"], window=case["window"], sinks=case["sinks"], frame=case["frame"])
    shift = scale = gate = None
    if s["modulation"] is not None:
        shift, scale, gate = s["modulation"].unbind(1)
    if s["residual"] is None:
        return {"y": ops.norm(s["x"], kind=case["kind"], weight=s["weight"], bias=s["bias"], scale=scale, shift=shift,
                              group=case["group"])}
    hidden, y = ops.residual_norm(s["x"], s["residual"], gate=gate, post_weight=s["post_weight"],
                                  residual_scale=case["residual_scale"], kind=case["kind"], weight=s["weight"], bias=s["bias"],
                                  scale=scale, shift=shift, group=case["group"])
    return {"hidden": hidden, "y": y}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------------------------------------- what a pass has to do


def _pairs_and_keys(case):
    """Visible (query, key) pairs of one head, and keys that some query of their stream sees."""
    pairs = keys = 0
    for n, kv in zip(*_lengths(case)):
        f = np.arange(kv - n, kv) // case["frame"]
        high = np.minimum((f + 1) * case["frame"], kv)
        low = np.maximum((f - case["window"] + 1) * case["frame"], 0)
        first = np.minimum(case["sinks"] * case["frame"], high)
        pairs += int((high - np.maximum(low, first) + first).sum())
        keys += int(high[-1] - max(low[0], first[-1]) + first[-1])
    return pairs, keys


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        n, pairs = case["tokens"], case["pairs_t"] + case["pairs_y"] + case["pairs_x"]
        return {"bytes": 2 * n * case["heads"] * case["head_dim"] * size + 12 * n + 8 * pairs, "flops": 6 * n * case["heads"] * pairs}
    if case["op"] == "append":
        n, pairs = sum(_lengths(case)[0]), case["pairs_t"] + case["pairs_y"] + case["pairs_x"]
        heads = case["q_heads"] + 2 * case["kv_heads"]
        return {"bytes": 2 * n * heads * case["head_dim"] * size + 12 * n + 8 * pairs,
                "flops": 6 * n * (case["q_heads"] + case["kv_heads"]) * pairs}
    if case["op"] == "attention":
        pairs, keys = _pairs_and_keys(case)
        n, d = sum(_lengths(case)[0]), case["head_dim"]
        return {"bytes": 2 * n * case["q_heads"] * d * size + 2 * keys * case["kv_heads"] * d * size,
                "flops": 4 * pairs * case["q_heads"] * d}
    n = case["rows"] * case["width"]
    vectors = 1 + (case["kind"] == "layer") + (case["residual"] and case["post"])
    if case["modulated"]:
        vectors += -(-case["rows"] // case["group"]) * (3 if case["residual"] else 2)
    return {"bytes": ((4 if case["residual"] else 2) * n + vectors * case["width"]) * size, "flops": 10 * n}


# --------------------------------------------------------------------------------------- definitions in 64 bits


def _exact_turn(x, positions, frequencies, case):
    """Each pair as a complex number, times the unit number of its angle."""
    counts = (case["pairs_t"], case["pairs_y"], case["pairs_x"])
    pairs = sum(counts)
    at = torch.cat([positions[:, a:a + 1].double().expand(-1, n) for a, n in enumerate(counts)], 1)
    unit = torch.polar(torch.ones_like(at), at * frequencies)[:, None]
    out = x.double().clone()
    if case["interleaved"]:
        z = torch.view_as_complex(out[..., :2 * pairs].reshape(*x.shape[:2], pairs, 2).contiguous()) * unit
        out[..., :2 * pairs] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(out[..., :pairs], out[..., pairs:2 * pairs]) * unit
        out[..., :pairs], out[..., pairs:2 * pairs] = z.real, z.imag
    return out


def _exact_attention(s):
    case = s["case"]
    d, page, ratio = case["head_dim"], case["page"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, kv) in enumerate(zip(*_lengths(case))):
        pages = s["table"][b, :-(-kv // page)].long()
        keys, values = (c[pages].flatten(0, 1)[:kv] for c in (s["k_cache"], s["v_cache"]))
        for lo in range(0, n, 2048):
            hi = min(n, lo + 2048)
            qf = (torch.arange(kv - n + lo, kv - n + hi, device="cuda") // case["frame"])[:, None]
            kf = (torch.arange(kv, device="cuda") // case["frame"])[None]
            hidden = (kf > qf) | ((kf <= qf - case["window"]) & (kf >= case["sinks"]))
            for h in range(case["q_heads"]):
                score = s["q"][at + lo:at + hi, h].double() @ keys[:, h // ratio].double().T / math.sqrt(d)
                p = torch.softmax(score.masked_fill(hidden, -math.inf), 1)
                out[at + lo:at + hi, h] = p @ values[:, h // ratio].double()
        at += n
    return out


def _exact_norm(s):
    case = s["case"]

    def unit(t):
        if case["kind"] == "layer":
            return (t - t.mean(1, keepdim=True)) / torch.sqrt(t.var(1, unbiased=False, keepdim=True) + 1e-6)
        return t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-6)

    x = s["x"].double()
    if s["modulation"] is not None:
        m = s["modulation"].double().repeat_interleave(case["group"], 0)[:case["rows"]]
    h = x
    if s["residual"] is not None:
        if s["post_weight"] is not None:
            x = unit(x) * s["post_weight"].double()
        h = case["residual_scale"] * s["residual"].double() + (x if s["modulation"] is None else m[:, 2] * x)
    y = unit(h) * s["weight"].double() + (0 if s["bias"] is None else s["bias"].double())
    if s["modulation"] is not None:
        y = y + y * m[:, 1] + m[:, 0]
    return {"y": y} if s["residual"] is None else {"hidden": h, "y": y}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_turn(s["x"], s["positions"], s["frequencies"], case)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "norm":
        return _exact_norm(s)
    hq, hk = case["q_heads"], case["kv_heads"]
    turned = _exact_turn(s["qkv"][:, :hq + hk], s["positions"], s["frequencies"], case)
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    at = 0
    for b, (n, kv) in enumerate(zip(*_lengths(case))):
        place = torch.arange(kv - n, kv, device="cuda")
        page = s["table"][b].long()[place // case["page"]]
        k_cache[page, place % case["page"]] = turned[at:at + n, hq:]
        v_cache[page, place % case["page"]] = s["qkv"][at:at + n, hq + hk:].double()
        at += n
    return {"q": turned[:, :hq], "k_cache": k_cache, "v_cache": v_cache}
