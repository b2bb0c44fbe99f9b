"""GPU: attention over a paged cache with a sliding window of frames and first frames that stay
visible, against the formula in FP64."""

from __future__ import annotations

import pytest
import torch

import token_reference as ref
from jasnamacos_b200.deform_conv import InvalidArgument, Unsupported

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from jasnamacos_b200.token_ops import CudaTokenOps

    return CudaTokenOps()


def normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def make(seed, lengths, steps, q_heads, heads, dim, page, dtype, padding=0, q_scale=1.5):
    """A step of queries and a cache of shuffled pages that holds NaN wherever no stream has a token."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [max(0, -(-n // page)) for n in lengths]
    total = sum(need) + 2
    order = torch.randperm(total, generator=g, device="cuda").int()
    table = torch.full((len(lengths), max(need + [1])), -1, dtype=torch.int32, device="cuda")
    k = torch.full((total, page, heads, dim), float("nan"), dtype=dtype, device="cuda")
    v = k.clone()
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        for c in (k, v):
            flat = torch.full((n * page, heads, dim), float("nan"), dtype=dtype, device="cuda")
            flat[:max(0, lengths[b])] = normal(g, (max(0, lengths[b]), heads, dim), dtype)
            c[table[b, :n].long()] = flat.view(n, page, heads, dim)
    starts = torch.tensor([sum(steps[:i]) for i in range(len(steps) + 1)], dtype=torch.int32, device="cuda")
    q = normal(g, (sum(steps) + padding, q_heads, dim), dtype, q_scale)
    return dict(q=q, k_cache=k, v_cache=v, table=table, starts=starts,
                lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))


def bounds(s):
    steps = s["starts"][1:] - s["starts"][:-1]
    return dict(max_q=int(steps.max()), max_kv=max(0, int(s["lengths"].max())))


def run(ops, s, **args):
    return ops.attention(**s, **bounds(s), **args)


def device_ok(ops):
    assert ops.lib.dcn_device_error() == 0


CASES = {
    # name: lengths, steps, q_heads, heads, head_dim, page, window, sinks, frame
    "one_key": ([1], [1], 1, 1, 64, 16, 1, 0, 1),
    "tokens": ([1, 2, 17, 130, 257, 1000], [1] * 6, 8, 2, 128, 16, 64, 4, 1),
    "tokens_long": ([5000, 3, 2047], [1, 1, 1], 16, 4, 128, 64, 4096, 16, 1),
    "tokens_many_heads": ([700, 90], [1, 1], 64, 1, 64, 32, 300, 0, 1),
    "tokens_ratio_128": ([300], [1], 128, 1, 64, 16, 1000, 0, 1),
    "ratio_3": ([61, 200, 640], [5, 41, 100], 6, 2, 128, 48, 50, 3, 1),
    "ratio_7_odd_heads": ([333, 129], [17, 129], 21, 3, 64, 16, 60, 0, 1),
    "causal": ([300, 128, 129, 1], [300, 128, 1, 1], 4, 4, 128, 128, 100000, 0, 1),
    "causal_chunk": ([1500, 700], [600, 257], 4, 2, 64, 256, 100000, 0, 1),
    "window_1": ([400], [400], 2, 2, 64, 16, 1, 0, 1),
    "window_sinks": ([2000, 1023], [513, 300], 4, 1, 128, 64, 129, 5, 1),
    "sinks_past_window": ([900], [700], 2, 2, 64, 64, 3, 400, 1),
    "frames": ([1280, 256, 512], [256, 256, 512], 4, 4, 64, 256, 3, 1, 256),
    "frames_odd": ([700, 77, 350], [140, 77, 1], 4, 2, 128, 48, 4, 2, 35),
    "frames_cut": ([1000], [333], 2, 2, 64, 16, 2, 1, 300),
    "frame_long": ([900], [100], 2, 1, 128, 64, 1, 0, 100000),
    "page_odd": ([500, 77], [60, 77], 4, 2, 64, 80, 100, 2, 3),
    "page_one_stream": ([700, 700], [128, 128], 4, 2, 128, 704, 2, 0, 128),
    "empty_streams": ([0, 40, 0, 300, 5], [0, 3, 0, 0, 5], 4, 2, 64, 16, 16, 1, 1),
    "more_queries_than_keys": ([10, 0, 200], [25, 4, 200], 4, 2, 64, 16, 30, 1, 1),
    "streams_70": (list(range(1, 71)), [k % 3 for k in range(70)], 2, 2, 64, 16, 20, 2, 1),
    "two_tiles": ([256], [256], 1, 1, 128, 64, 1000, 0, 1),
    # more row blocks than SMs, the last ones split: one and several tokens a stream, one stream without keys
    "tokens_tail": ([300 + 37 * k for k in range(40)], [1] * 40, 8, 4, 64, 32, 900, 3, 1),
    "tokens_tail_steps": ([0] + [1500 + 11 * k for k in range(54)], [2] + [1 + k % 5 for k in range(54)], 3, 3, 128, 64, 700, 0, 1),
    "four_tiles_long": ([3000], [600], 2, 1, 128, 64, 500, 100, 1),
}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", list(CASES))
def test_attention(ops, name, dtype):
    lengths, steps, q_heads, heads, dim, page, window, sinks, frame = CASES[name]
    s = make(len(name) + sum(lengths), lengths, steps, q_heads, heads, dim, page, dtype)
    args = dict(window=window, sinks=sinks, frame=frame)
    want, bound = ref.attention(**s, **args)
    out = run(ops, s, **args)
    ref.check(out, want, bound)
    assert torch.equal(run(ops, s, **args), out)  # the same bits every time
    device_ok(ops)


@pytest.mark.parametrize("dtype,dim", [(F32, 64), (F32, 128), (F32, 33), (F16, 80), (BF16, 256), (F16, 8), (BF16, 1)])
@pytest.mark.parametrize("name", ["tokens", "ratio_3", "window_sinks", "frames_odd", "empty_streams", "more_queries_than_keys"])
def test_attention_other_types_and_heads(ops, name, dtype, dim):
    lengths, steps, q_heads, heads, _, page, window, sinks, frame = CASES[name]
    s = make(dim, lengths, steps, q_heads, heads, dim, page, dtype)
    want, bound = ref.attention(**s, window=window, sinks=sinks, frame=frame)
    ref.check(run(ops, s, window=window, sinks=sinks, frame=frame), want, bound)


@pytest.mark.parametrize("page", [1, 3, 17, 24, 100])
def test_attention_other_pages(ops, page):
    s = make(page, [300, 41], [40, 41], 4, 2, 64, page, F16)
    want, bound = ref.attention(**s, window=90, sinks=2)
    ref.check(run(ops, s, window=90, sinks=2), want, bound)


@pytest.mark.parametrize("scale", [0.0, 0.02, 1.0, -0.125])
def test_attention_scale(ops, scale):
    """Flat, sharp and negated scores; scale 0 is the mean of the visible values."""
    s = make(4, [700, 150], [40, 1], 4, 2, 64, 64, F16)
    want, bound = ref.attention(**s, window=400, scale=scale)
    ref.check(run(ops, s, window=400, scale=scale), want, bound)


@pytest.mark.parametrize("steps", [[1], [200]])
def test_attention_growing_scores(ops, steps):
    """Each tile's scores exceed all before it by far (the running maximum moves every time), or fall."""
    s = make(5, [900], steps, 2, 2, 64, 64, BF16)
    ramp = torch.linspace(0.5, 12.0, 960, device="cuda").view(-1, 64, 1, 1).to(BF16)
    for direction in (1, -1):
        t = dict(s)
        rows = s["table"][0].long()
        k = s["k_cache"].clone()
        k[rows] = (ramp if direction == 1 else ramp.flip(0).flip(1)) * 1.0
        t["k_cache"] = k
        t["q"] = s["q"].abs()
        want, bound = ref.attention(**t, window=10000)
        ref.check(run(ops, t, window=10000), want, bound)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("steps,frame", [([1, 1], 1), ([300, 3], 1), ([384, 128], 64)])
def test_attention_hidden_non_finite(ops, steps, frame, dtype):
    """A key or value that a row does not see leaves that row alone, whatever it holds; one that it sees shows."""
    s = make(6, [640, 512], steps, 4, 2, 64, 64, dtype)
    args = dict(window=128 // frame, sinks=1, frame=frame)
    want, bound = ref.attention(**s, **args)
    ids = s["table"][0].long()
    k, v = s["k_cache"].clone(), s["v_cache"].clone()
    for c, at, value in ((k, 520, float("nan")), (v, 530, float("inf")), (v, 300, float("nan")), (k, 300, float("inf")),
                         (v, 639, float("nan")), (k, 200, float("-inf")), (v, 210, float("-inf"))):
        c[ids[at // 64], at % 64, 1] = value
    t = dict(s, k_cache=k, v_cache=v)
    out = run(ops, t, **args)
    position = torch.arange(640 - steps[0], 640, device="cuda")[:, None]
    spoiled = torch.tensor([520, 530, 300, 639, 200, 210], device="cuda")[None]
    hit = ref.visible(position, spoiled, args["window"], args["sinks"], frame).any(1)
    clean = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
    clean[:steps[0], 2:] = ~hit[:, None]
    ref.check(out[clean], want[clean], bound[clean])
    assert not bool(torch.isfinite(out[~clean]).any())


def test_attention_rows_of_infinity(ops):
    """A row whose query is not finite is not finite; the others do not notice."""
    s = make(7, [300], [150], 2, 2, 64, 64, F16)
    want, bound = ref.attention(**s, window=1000)
    s["q"][7, 0] = float("nan")
    s["q"][90, 1, 5] = float("inf")
    out = run(ops, s, window=1000)
    clean = torch.ones(150, 2, dtype=torch.bool, device="cuda")
    clean[7, 0] = clean[90, 1] = False
    ref.check(out[clean], want[clean], bound[clean])
    assert not bool(torch.isfinite(out[7, 0]).any())


@pytest.mark.parametrize("steps", [[1, 1, 1], [70, 1, 200]])
def test_attention_strides(ops, steps):
    """Queries inside a wider projection, keys and values of a page side by side with heads before slots,
    a table inside a wider one, padding rows that belong to no stream, a given result."""
    s = make(8, [500, 64, 333], steps, 4, 2, 128, 64, F16, padding=5)
    want, bound = ref.attention(**s, window=200, sinks=3)
    t = dict(s)
    wide = torch.zeros(s["q"].shape[0], 9, 128, dtype=F16, device="cuda")
    wide[:, 3:7] = s["q"]
    t["q"] = wide[:, 3:7]
    pages, page, heads, dim = s["k_cache"].shape
    both = torch.empty(pages, heads, 2, page, dim, dtype=F16, device="cuda")
    both[:, :, 0], both[:, :, 1] = s["k_cache"].transpose(1, 2), s["v_cache"].transpose(1, 2)
    t["k_cache"], t["v_cache"] = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    table = torch.full((3, 31), -7, dtype=torch.int32, device="cuda")
    table[:, :s["table"].shape[1]] = s["table"]
    t["table"] = table[:, :s["table"].shape[1]]
    out = torch.full((s["q"].shape[0], 11, 128), 3.0, dtype=F16, device="cuda")
    view = out[:, 5:9]
    assert run(ops, t, window=200, sinks=3, out=view) is view
    n = sum(steps)
    ref.check(view[:n], want[:n], bound[:n])
    assert bool((out[n:] == 3).all()) and bool((out[:, :5] == 3).all()) and bool((out[:, 9:] == 3).all())
    # elements off 16-byte alignment
    odd = torch.zeros(s["q"].shape[0], 4, 129, dtype=F16, device="cuda")
    odd[..., 1:] = s["q"]
    ref.check(run(ops, dict(t, q=odd[..., 1:]), window=200, sinks=3)[:n], want[:n], bound[:n])


@pytest.mark.parametrize("steps", [[1, 1], [300, 2]])
def test_attention_past_32_bits(ops, steps):
    """Pages past element 2^31 of the cache."""
    s = make(9, [320, 200], steps, 4, 2, 128, 64, F16)
    want, bound = ref.attention(**s, window=10000)
    pages = 140000
    k = torch.empty(pages, 64, 2, 128, dtype=F16, device="cuda")  # 2.3e9 elements each
    v = torch.empty_like(k)
    table = s["table"].clone()
    for b in range(2):
        for c in range(table.shape[1]):
            if table[b, c] >= 0:
                k[pages - 1 - table[b, c]], v[pages - 1 - table[b, c]] = s["k_cache"][table[b, c]], s["v_cache"][table[b, c]]
                table[b, c] = pages - 1 - table[b, c]
    ref.check(run(ops, dict(s, k_cache=k, v_cache=v, table=table), window=10000), want, bound)


def test_attention_bounds_are_only_hints(ops):
    """Smaller and larger max_q and max_kv than the streams have: the same result to its bound."""
    s = make(10, [2000, 600], [300, 20], 4, 2, 64, 64, F16)
    want, bound = ref.attention(**s, window=700, sinks=2)
    for max_q, max_kv in ((300, 2000), (1000, 100000), (300, 0), (300, 10), (1, 2000), (0, 0), (20, 600)):
        ref.check(ops.attention(**s, max_q=max_q, max_kv=max_kv, window=700, sinks=2), want, bound)


def test_attention_other_stream_and_graph(ops):
    s = make(11, [900, 77, 300], [1, 1, 1], 8, 2, 128, 16, BF16)
    want, bound = ref.attention(**s, window=500)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = run(ops, s, window=500, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    ref.check(out, want, bound)
    out = torch.zeros_like(out)
    graph = torch.cuda.CUDAGraph()
    limits = bounds(s)
    with torch.cuda.graph(graph):
        ops.attention(**s, **limits, window=500, out=out)
    s["q"].mul_(-1)
    want, bound = ref.attention(**s, window=500)
    graph.replay()
    ref.check(out, want, bound)


def test_attention_refused(ops):
    s = make(12, [100], [10], 4, 2, 64, 16, F16)
    assert run(ops, dict(s, q=s["q"][:0], starts=torch.zeros_like(s["starts"])), window=4).shape == (0, 4, 64)
    good = dict(s, max_q=10, max_kv=100, window=4)
    for bad in (dict(window=0), dict(sinks=-1), dict(frame=0), dict(scale=float("nan")), dict(q=s["q"].bfloat16()),
                dict(q=s["q"][..., :32]), dict(table=s["table"].long()), dict(lengths=s["lengths"].cpu()), dict(starts=s["starts"][:1]),
                dict(out=s["q"][:, :2]), dict(q=s["q"][0]), dict(v_cache=s["v_cache"].bfloat16())):
        with pytest.raises(InvalidArgument):
            ops.attention(**(good | bad))
    with pytest.raises(Exception):
        ops.attention(**(good | dict(q=s["q"][:, :3])))  # 3 query heads over 2 key heads
    with pytest.raises(Unsupported):
        big = make(12, [20], [10], 4, 2, 264, 16, F16)
        run(ops, big, window=4)
    need = ops.attention_workspace_bytes(**good)
    if need:
        with pytest.raises(InvalidArgument):
            ops.attention(**good, workspace=torch.empty(need - 16, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("lengths,steps", [([2000, 600], [300, 20]), ([700] * 40, [1] * 40), ([900] + [50] * 200, [600] + [1] * 200)])
def test_attention_without_known_limits(ops, lengths, steps):
    """The largest max_q, max_kv and window there are: the launch follows the tensors."""
    s = make(13, lengths, steps, 4, 2, 64, 64, F16)
    want, bound = ref.attention(**s, window=5000)
    most = 2**31 - 1
    ref.check(ops.attention(**s, max_q=most, max_kv=most, window=most), want, bound)


@pytest.mark.parametrize("name", ["max_q", "max_kv", "window", "sinks", "frame"])
def test_attention_counts_past_32_bits_are_refused(ops, name):
    s = make(14, [100], [10], 4, 2, 64, 16, F16)
    with pytest.raises(InvalidArgument):
        ops.attention(**(dict(s, max_q=10, max_kv=100, window=4) | {name: 2**32 + 4}))


@pytest.mark.parametrize("length,step,at", [(131000, 300, 130900), (262143, 4, 262141)])
def test_attention_long_rows_beside_non_finite_values(ops, length, step, at):
    """A value that only a step's last rows see, over a long cache: its rows are done one by one, no wait runs
    out meanwhile, and the rows before it are the formula's."""
    s = make(15, [length], [step], 2, 1, 64, 64, F16)
    want, bound = ref.attention(**s, window=10**6)
    v = s["v_cache"].clone()
    v[s["table"][0, at // 64].long(), at % 64, 0, 3] = float("inf")
    out = run(ops, dict(s, v_cache=v), window=10**6)
    torch.cuda.synchronize()
    device_ok(ops)
    clean = torch.arange(length - step, length, device="cuda") < at
    ref.check(out[clean], want[clean], bound[clean])
    assert not bool(torch.isfinite(out[~clean][..., 3]).any())
