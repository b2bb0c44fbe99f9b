"""GPU: calls of the token operators at the edges of what they promise, against the formulas in FP64."""

from __future__ import annotations

import math
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest
import torch

import token_reference as ref
from jasnamacos_b200 import _native
from jasnamacos_b200.deform_conv import InvalidArgument, InvalidShape, Unsupported

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
REPO = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def ops():
    from jasnamacos_b200.token_ops import CudaTokenOps

    return CudaTokenOps()


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def paged(gen, lengths, heads, dim, page, dtype):
    """A cache of shuffled pages full of values, and the streams' table (-1 where a stream has no page)."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + 2
    order = torch.randperm(total, generator=gen, device="cuda").int()
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return normal(gen, (total, page, heads, dim), dtype), normal(gen, (total, page, heads, dim), dtype), table


# ---- tokens before the first stream's ------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("lead,steps,lengths", [(5, [3, 4], [40, 9]), (3000, [3500, 2600], [9000, 4000])])
def test_append_leaves_out_tokens_before_the_first_stream(ops, dtype, lead, steps, lengths):
    """starts may begin past 0, as a slice of a larger batch's does: the tokens before it are no stream's.  Few
    tokens, and enough for the kernel that copies rows whole."""
    g = generator(lead)
    k_cache, v_cache, table = paged(g, lengths, 4, 128, 64, dtype)
    starts = ints([lead, lead + steps[0], lead + sum(steps)])
    k, v = (normal(g, (lead + sum(steps) + 2, 4, 128), dtype) for _ in range(2))
    want_k, want_v = k_cache.clone(), v_cache.clone()
    for b, n in enumerate(lengths):
        at = torch.arange(n - steps[b], n, device="cuda")
        page = table[b].long()[at // 64]
        lo = int(starts[b])
        want_k[page, at % 64], want_v[page, at % 64] = k[lo:lo + steps[b]], v[lo:lo + steps[b]]
    ops.append(k, v, k_cache, v_cache, table, starts, ints(lengths))
    assert torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("steps,lengths,split", [([1, 3], [40, 9], False), ([1, 2], [5000, 30], True),
                                                 ([300, 2], [300, 30], False), ([300, 7], [5000, 60], True)])
def test_attention_leaves_out_tokens_before_the_first_stream(ops, dtype, steps, lengths, split):
    """Rows of no stream keep what the result held, whichever kernel runs and whether its keys are split."""
    g = generator(sum(lengths))
    k_cache, v_cache, table = paged(g, lengths, 1, 64, 64, dtype)
    lead = 9
    starts = ints([lead, lead + steps[0], lead + sum(steps)])
    q = normal(g, (lead + sum(steps) + 2, 2, 64), dtype, 1.5)
    s = dict(q=q, k_cache=k_cache, v_cache=v_cache, table=table, starts=starts, lengths=ints(lengths))
    limits = dict(max_q=max(steps), max_kv=max(lengths), window=10000)
    assert (ops.attention_workspace_bytes(**s, **limits) > 0) == (split and dtype == F16)
    out = torch.full_like(q, 3.0)
    ops.attention(**s, **limits, out=out)
    want, bound = ref.attention(**s, window=10000)
    end = lead + sum(steps)
    ref.check(out[lead:end], want[lead:end], bound[lead:end])
    assert bool((out[:lead] == 3).all()) and bool((out[end:] == 3).all())


# ---- FP16 weights far below the largest ------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("streams,step,heads", [(1, 9472, 4), (4, 1, 37)])
def test_attention_many_small_weights(ops, dtype, streams, step, heads):
    """One key of weight 1, met first, whose value is 0, and 262,143 of weight 2^-25.1, whose values are 1 and make
    up the result.  All rows see all keys, and there are enough rows that no further launch splits them.

    Bound, of the result: a rounding of it and of the weights; a product's cut at 2^-25 of the sum it is added to, of
    each key; the chain of FP32 sums, two a tile of 128 keys.  And FP16 has weights of this size in multiples of
    2^-31: half of one, of each key."""
    keys, dim, page = 262144, 64, 1024
    q = torch.zeros(streams * step, heads, dim, dtype=dtype, device="cuda")
    q[..., 0] = 17.40625
    k = torch.zeros(keys // page, page, heads, dim, dtype=dtype, device="cuda")
    k[0, 0, :, 0] = 1.0
    v = torch.ones_like(k)
    v[0, 0] = 0.0
    s = dict(q=q, k_cache=k, v_cache=v, table=torch.arange(keys // page, device="cuda").int().expand(streams, -1).contiguous(),
             starts=ints([step * b for b in range(streams + 1)]), lengths=ints([keys] * streams), max_q=step, max_kv=keys,
             window=1, frame=1 << 20)
    assert ops.attention_workspace_bytes(**s) == 0
    rest = (keys - 1) * math.exp(-q[0, 0, 0].item())
    want = rest / (rest + 1)
    bound = want * (2 * ref.U[dtype] + keys * 2.0 ** -25 + keys / 64 * 2.0 ** -24) + (keys * 2.0 ** -32 if dtype == F16 else 0)
    off = (ops.attention(**s, scale=1.0).double() - want).abs().max().item()
    assert off <= bound, f"off by {off:.3g}, bound {bound:.3g}"


# ---- scales near zero ------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("steps", [[1, 2], [200, 3]])
@pytest.mark.parametrize("scale", [2.0 ** -104, -2.0 ** -104, 0.0])
def test_attention_small_scale_of_large_products(ops, dtype, steps, scale):
    """Queries and keys of 2^52: their products times the scale are ordinary scores."""
    g = generator(21)
    k_cache, v_cache, table = paged(g, [700, 150], 2, 64, 64, dtype)
    s = dict(q=normal(g, (sum(steps), 4, 64), dtype, 2.0 ** 51), k_cache=k_cache * 2.0 ** 52, v_cache=v_cache, table=table,
             starts=ints([0, steps[0], sum(steps)]), lengths=ints([700, 150]))
    want, bound = ref.attention(**s, window=400, scale=scale)
    ref.check(ops.attention(**s, max_q=max(steps), max_kv=700, window=400, scale=scale), want, bound)


# ---- rows done alone, item after item --------------------------------------------------------


def test_attention_rows_alone_beside_short_steps(ops):
    """A block takes a step of two row tiles, one of a single tile, and again one of two, each with a value that is
    not finite and that only the last rows see: each item's rows are done alone on its own account."""
    n, dim = 148, 64
    steps = [200] * n + [100] * n + [200] * n
    lengths = [264] * (3 * n)
    g = generator(22)
    k_cache, v_cache, table = paged(g, lengths, 1, dim, 24, F16)
    starts = ints([sum(steps[:b]) for b in range(3 * n + 1)])
    s = dict(q=normal(g, (sum(steps), 1, dim), F16, 1.5), k_cache=k_cache, v_cache=v_cache, table=table, starts=starts,
             lengths=ints(lengths))
    want, bound = ref.attention(**s, window=10000)
    v = v_cache.clone()
    v[table[:, 260 // 24].long(), 260 % 24, 0, 5] = float("inf")
    out = ops.attention(**dict(s, v_cache=v), max_q=200, max_kv=264, window=10000)
    stream = torch.repeat_interleave(torch.arange(3 * n, device="cuda"), torch.tensor(steps, device="cuda"))
    position = 264 - starts.long()[stream + 1] + torch.arange(sum(steps), device="cuda")
    clean = position < 260
    ref.check(out[clean], want[clean], bound[clean])
    assert not bool(torch.isfinite(out[~clean][..., 5]).any())
    other = torch.arange(dim, device="cuda") != 5
    ref.check(out[..., other], want[..., other], bound[..., other])
    assert ops.lib.dcn_device_error() == 0


# ---- sizes past 32 bits ----------------------------------------------------------------------


def test_sizes_past_32_bits_are_refused(ops):
    """Refused, not cut to their low bits: here 64 elements of a row, one head, one page."""
    wide = torch.zeros(1, 2 ** 32 + 64, dtype=F16, device="cuda")
    with pytest.raises(Unsupported):
        ops.norm(wide, out=wide)
    with pytest.raises(Unsupported):
        ops.residual_norm(wide, wide, hidden=wide, out=wide)
    x = wide[:, :64].view(1, 1, 64).expand(1, 2 ** 32 + 1, 64)
    at, f = torch.zeros(1, 3, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.float64, device="cuda")
    with pytest.raises(InvalidShape):
        ops.rotary(x, at, f, (1, 0, 0), out=x)
    cache = torch.zeros(1, 16, 1, 64, dtype=F16, device="cuda")
    many_pages = cache.expand(2 ** 32 + 1, 16, 1, 64)
    long_page = cache[:, :1].expand(1, 2 ** 32 + 1, 1, 64)
    row = torch.zeros(1, 1, 64, dtype=F16, device="cuda")
    for pages in (many_pages, long_page):
        s = dict(k_cache=pages, v_cache=pages, table=ints([[0]]), starts=ints([0, 1]), lengths=ints([1]))
        with pytest.raises(InvalidArgument):
            ops.append(row, row, **s)
        with pytest.raises(InvalidArgument):
            ops.attention(row, **s, max_q=1, max_kv=1, window=1)
    s = dict(k_cache=cache, v_cache=cache, table=ints([[0]]), starts=ints([0, 1]), lengths=ints([1]))
    with pytest.raises(InvalidShape):
        ops.append(row, row, **s, q=x, q_out=x)
    with pytest.raises(InvalidShape):
        ops.attention(x, **s, max_q=1, max_kv=1, window=1, out=x)


# ---- set-up of one operator and the others ---------------------------------------------------


def test_convolution_does_not_depend_on_the_token_operators(tmp_path):
    """Where the set-up of the attention and norm kernels fails, as it would with kernels that a device refuses, those
    operators say so and the others run.  The failure is a stand-in for the two set-up functions, loaded ahead of them."""
    fake = tmp_path / "fake.cpp"
    fake.write_text("namespace dcn {\nint token_attention_prepare_device() { return 9; }  // invalid configuration\n"
                    "int token_norm_prepare_device() { return 9; }\n}\n")
    lib = tmp_path / "libfake.so"
    subprocess.run(["g++", "-shared", "-fPIC", "-o", str(lib), str(fake)], check=True)
    code = f"""
        import ctypes, sys
        sys.path.insert(0, {str(REPO)!r})
        ctypes.CDLL({str(lib)!r}, mode=ctypes.RTLD_GLOBAL)
        import torch
        from jasnamacos_b200 import synthetic
        from jasnamacos_b200.deform_conv import CommandFailed, CudaDeformConv
        from jasnamacos_b200.token_ops import CudaTokenOps
        inp = synthetic.generate(1)
        out = CudaDeformConv().run_float16(inp.shape, inp.input, inp.offset, inp.mask, inp.weight, inp.bias)
        print("convolution", out.size)
        ops = CudaTokenOps()
        x = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda")
        at, f = torch.zeros(4, 3, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.float64, device="cuda")
        ops.rotary(x, at, f, (1, 0, 0))
        print("rotary")
        cache = torch.zeros(1, 16, 2, 64, dtype=torch.float16, device="cuda")
        one = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
        s = dict(k_cache=cache, v_cache=cache, table=one[None, :1].contiguous(), starts=one, lengths=one[1:])
        ops.append(x, x, **s)
        limits = dict(max_q=4, max_kv=4, window=4)
        ops.attention(x.float(), **dict(s, k_cache=cache.float(), v_cache=cache.float()), **limits)
        print("attention on CUDA cores")
        for name, call in (("attention", lambda: ops.attention(x, **s, **limits)), ("norm", lambda: ops.norm(x.view(4, 128)))):
            for again in range(2):
                try:
                    call()
                except CommandFailed:
                    print(name, "refused")
        torch.cuda.synchronize()
    """
    done = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    said = done.stdout.split("\n")
    assert said[1:-1] == ["rotary", "attention on CUDA cores"] + ["attention refused"] * 2 + ["norm refused"] * 2, done.stdout


def test_first_call_of_an_operator_may_be_captured():
    """In a process that has launched other operators: the set-up of attention and norm is no stream operation."""
    code = f"""
        import sys
        sys.path.insert(0, {str(REPO)!r})
        import torch
        from jasnamacos_b200.token_ops import CudaTokenOps
        ops = CudaTokenOps()
        x = torch.randn(512, 2, 64, device="cuda").half()
        at, f = torch.zeros(512, 3, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.float64, device="cuda")
        ops.rotary(x, at, f, (1, 0, 0))
        cache = torch.randn(1, 512, 2, 64, device="cuda").half()
        one = torch.tensor([0, 512], dtype=torch.int32, device="cuda")
        s = dict(k_cache=cache, v_cache=cache, table=one[None, :1].contiguous(), starts=one, lengths=one[1:])
        rows = torch.randn(9001, 512, device="cuda").half()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = ops.attention(x, **s, max_q=512, max_kv=512, window=512)
            n = ops.norm(rows)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ops.attention(x, **s, max_q=512, max_kv=512, window=512)) and torch.equal(n, ops.norm(rows))
        assert bool(a.isfinite().all()) and bool(n.isfinite().all()) and bool(n.any())
    """
    done = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


# ---- keys without a page ---------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("steps", [[1, 2, 1], [300, 3, 200], [33, 3, 40]])
@pytest.mark.parametrize("spoiled", [False, True])
def test_attention_keys_without_a_page_are_zeros(ops, dtype, steps, spoiled):
    """Visible positions whose page id is outside the cache, or that lie past the table, have a key and a value of
    zeros; also for rows that are done alone beside a value that is not finite."""
    g = generator(23)
    lengths, page = [900, 130, 500], 64
    k_cache, v_cache, table = paged(g, lengths, 2, 64, page, dtype)
    pages = k_cache.shape[0]
    table[0, 3], table[0, 7], table[1, 0], table[2, 2] = -1, pages, -(2 ** 31), 2 ** 31 - 1
    cut = table[:, :12].contiguous()  # stream 0 runs on for 132 positions more
    s = dict(q=normal(g, (sum(steps), 4, 64), dtype, 1.5), k_cache=k_cache, v_cache=v_cache, table=cut,
             starts=ints([0, steps[0], steps[0] + steps[1], sum(steps)]), lengths=ints(lengths))
    full = torch.full((3, 15), pages, dtype=torch.int32, device="cuda")  # the reference has a page of zeros there
    full[:, :12] = torch.where((cut >= 0) & (cut < pages), cut, pages)
    zeros = torch.zeros_like(k_cache[:1])
    t = dict(s, k_cache=torch.cat([k_cache, zeros]), v_cache=torch.cat([v_cache, zeros]), table=full)
    want, bound = ref.attention(**t, window=600, sinks=70)
    clean = torch.ones(sum(steps), dtype=torch.bool, device="cuda")
    if spoiled:
        at = 497  # of stream 2, which only the rows from it on see
        s["v_cache"] = v_cache.clone()
        s["v_cache"][table[2, at // page].long(), at % page, :, 7] = float("nan")
        clean[steps[0] + steps[1]:] = torch.arange(500 - steps[2], 500, device="cuda") < at
    out = ops.attention(**s, max_q=max(steps), max_kv=900, window=600, sinks=70)
    ref.check(out[clean], want[clean], bound[clean])
    assert bool(out[~clean][..., 7].isnan().all())
    other = torch.arange(64, device="cuda") != 7
    ref.check(out[..., other], want[..., other], bound[..., other])


# ---- a caller's own scratch ------------------------------------------------------------------


@pytest.mark.parametrize("steps", [[1], [300]])
def test_attention_workspace_of_the_caller(ops, steps):
    g = generator(24)
    k_cache, v_cache, table = paged(g, [5000], 2, 64, 64, F16)
    s = dict(q=normal(g, (steps[0], 4, 64), F16, 1.5), k_cache=k_cache, v_cache=v_cache, table=table, starts=ints([0, steps[0]]),
             lengths=ints([5000]))
    want, bound = ref.attention(**s, window=10000)
    limits = dict(max_q=steps[0], max_kv=5000, window=10000)
    need = ops.attention_workspace_bytes(**s, **limits)
    assert need > 0
    guarded = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    out = ops.attention(**s, **limits, workspace=guarded[:need])
    ref.check(out, want, bound)
    assert bool((guarded[need:] == 0xA5).all())
    kept = out.clone()
    for bad in (guarded[:need - 16], guarded[1:need + 1], guarded[:0], guarded[::2], torch.zeros(need, dtype=torch.uint8)):
        with pytest.raises(InvalidArgument):
            ops.attention(**s, **limits, workspace=bad, out=out)
    assert torch.equal(out, kept)
    three = dict(s, q=s["q"][:, :3])  # three query heads over two key heads
    with pytest.raises(InvalidShape):
        ops.attention(**three, **limits)


def test_attention_on_two_streams_at_once(ops):
    """One object, two CUDA streams, calls that split their keys: each has its own scratch."""
    g = generator(25)
    k_cache, v_cache, table = paged(g, [20000, 9000], 2, 128, 64, BF16)
    calls = []
    for seed in range(2):
        s = dict(q=normal(g, (2, 8, 128), BF16, 1.5), k_cache=k_cache, v_cache=v_cache, table=table, starts=ints([0, 1, 2]),
                 lengths=ints([20000, 9000]), max_q=1, max_kv=20000, window=30000)
        assert ops.attention_workspace_bytes(**s) > 0
        calls.append((s, ops.attention(**s)))
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(50):
        for i, side in enumerate(sides):
            got[i].append(ops.attention(**calls[i][0], stream=side))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, calls[i][1]) for o in got[i])


# ---- results that a caller leaves out ----------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,width,post", [(3, 1155, False), (40, 1024, True), (9001, 512, False), (9001, 512, True)])
def test_norm_with_one_result(ops, dtype, rows, width, post):
    """The C entry with hidden alone and with out alone: the same bits as with both."""
    g = generator(rows + width)
    x, residual = normal(g, (rows, width), dtype), normal(g, (rows, width), dtype)
    weight = 1 + normal(g, (width,), dtype, 0.1)
    hidden, out = ops.residual_norm(x, residual, post_weight=weight if post else None, residual_scale=0.5)
    for keep in ("hidden", "out"):
        result = torch.full_like(x, 3.0)
        at = weight.data_ptr() if post else None
        args = _native.DcnTokenNormArgs(
            rows=rows, group=rows, width=width, dtype=_native.DCN_DTYPE_F32 if dtype == F32 else _native.DCN_DTYPE_F16,
            kind=_native.DCN_NORM_RMS, post=int(post), epsilon=1e-6, residual_scale=0.5, x=x.data_ptr(),
            residual=residual.data_ptr(), post_weight=at, x_stride=width, residual_stride=width, hidden_stride=width,
            out_stride=width, **{keep: result.data_ptr()})
        assert ops.lib.dcn_token_norm(args, torch.cuda.current_stream().cuda_stream or None) == _native.DCN_OK
        assert torch.equal(result, hidden if keep == "hidden" else out)
