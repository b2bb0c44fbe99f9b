"""GPU: the norms around a block, the rotary positions and the cache append against FP64 formulas."""

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


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------------------- norm


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (5, 64), (2, 257), (37, 512), (9, 1000), (4, 1155), (6, 2048),
                                        (3, 4104), (2, 8192), (2, 8191)])
def test_norm_before_a_block(ops, dtype, kind, rows, width):
    g = generator(rows * 10007 + width)
    x = normal(g, (rows, width), dtype, 2.0) + 1
    w, b = 1 + normal(g, (width,), dtype, 0.2), normal(g, (width,), dtype, 0.2)
    scale, shift = normal(g, (-(-rows // 2), width), dtype, 0.3), normal(g, (-(-rows // 2), width), dtype, 0.3)
    ref.check(ops.norm(x, kind=kind), *ref.norm(x, kind=kind)[1])
    ref.check(ops.norm(x, kind=kind, weight=w, bias=b), *ref.norm(x, kind=kind, weight=w, bias=b)[1])
    ref.check(ops.norm(x, kind=kind, weight=w, scale=scale, shift=shift, group=2, eps=1e-3),
              *ref.norm(x, kind=kind, weight=w, scale=scale, shift=shift, group=2, eps=1e-3)[1])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("rows,width,group", [(1, 64, 1), (7, 96, 3), (130, 1024, 64), (5, 1155, 5), (3, 5000, 2)])
def test_residual_norm(ops, dtype, kind, post, rows, width, group):
    g = generator(rows * 7919 + width)
    groups = -(-rows // group)
    x, residual = normal(g, (rows, width), dtype, 2.0) - 0.5, normal(g, (rows, width), dtype, 3.0)
    # shift, scale and gate of a group lie side by side, as one projection gives them
    shift, scale, gate = normal(g, (groups, 3, width), dtype, 0.4).unbind(1)
    args = dict(gate=gate, residual_scale=0.75, kind=kind, weight=1 + normal(g, (width,), dtype, 0.1), scale=scale, shift=shift,
                group=group)
    if post:
        args |= dict(post_weight=1 + normal(g, (width,), dtype, 0.1), post_bias=normal(g, (width,), dtype, 0.1))
    hidden, out = ops.residual_norm(x, residual, **args)
    want_hidden, want_out = ref.norm(x, residual, **args)
    ref.check(hidden, *want_hidden)
    ref.check(out, *want_out)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("width,group,post", [(64, 1000, False), (512, 47, True), (1000, 64, False), (1024, 256, True)])
def test_residual_norm_of_many_rows(ops, dtype, kind, width, group, post):
    """Enough rows for the kernel that folds a group's vectors once a block; groups that end inside a block."""
    rows = 20011
    g = generator(width + group)
    groups = -(-rows // group)
    x, residual = normal(g, (rows, width), dtype, 2.0) - 0.5, normal(g, (rows, width), dtype, 3.0)
    shift, scale, gate = normal(g, (groups, 3, width), dtype, 0.4).unbind(1)
    args = dict(gate=gate, residual_scale=1.25, kind=kind, weight=1 + normal(g, (width,), dtype, 0.1), scale=scale, shift=shift,
                group=group, bias=normal(g, (width,), dtype, 0.1))
    if post:
        args |= dict(post_weight=1 + normal(g, (width,), dtype, 0.1), post_bias=normal(g, (width,), dtype, 0.1))
    hidden, out = ops.residual_norm(x, residual, **args)
    want_hidden, want_out = ref.norm(x, residual, **args)
    ref.check(hidden, *want_hidden)
    ref.check(out, *want_out)
    again = x.clone()
    ops.residual_norm(again, residual, **args, hidden=residual, out=again)  # in place
    assert torch.equal(residual, hidden) and torch.equal(again, out)
    ref.check(ops.norm(x, kind=kind, weight=args["weight"]), *ref.norm(x, kind=kind, weight=args["weight"])[1])
    spoiled = x.clone()
    spoiled[777, 3] = float("nan")
    clean = torch.arange(rows, device="cuda") != 777
    assert torch.equal(ops.norm(spoiled, kind=kind)[clean], ops.norm(x, kind=kind)[clean])


def test_norm_strides_and_in_place(ops):
    g = generator(5)
    wide = normal(g, (20, 3, 136), F16)
    x, residual = wide[:, 1, :128], wide[:, 2, 1:129]  # rows apart, the second one off 16-byte alignment
    want_hidden, want_out = ref.norm(x, residual, kind="layer")
    hidden, out = ops.residual_norm(x, residual, kind="layer")
    ref.check(hidden, *want_hidden)
    ref.check(out, *want_out)
    again = wide.clone()
    ops.residual_norm(again[:, 1, :128], again[:, 2, 1:129], kind="layer", hidden=again[:, 2, 1:129], out=again[:, 1, :128])
    assert torch.equal(again[:, 2, 1:129], hidden) and torch.equal(again[:, 1, :128], out)
    assert torch.equal(again[:, 0], wide[:, 0]) and torch.equal(again[:, 1, 128:], wide[:, 1, 128:])
    row = normal(g, (1, 64), F32)
    ref.check(ops.norm(row.expand(9, 64)), *ref.norm(row.expand(9, 64))[1])


def test_norm_special_rows(ops):
    x = torch.zeros(6, 64, dtype=F16, device="cuda")
    x[1] = 65504.0   # the squares' sum is far outside FP16
    x[2, 3] = float("nan")
    x[3, 5] = float("inf")
    x[4] = -7.0
    x[5] = torch.arange(64, device="cuda").half()
    rms, layer = ops.norm(x, kind="rms"), ops.norm(x, kind="layer")
    assert torch.equal(rms[0], torch.zeros(64, dtype=F16, device="cuda")) and torch.equal(layer[0], rms[0])
    assert torch.equal(rms[1], torch.ones(64, dtype=F16, device="cuda"))
    assert torch.equal(layer[1], torch.zeros(64, dtype=F16, device="cuda")) and torch.equal(layer[4], layer[1])
    assert bool(rms[2].isnan().all()) and bool(layer[2].isnan().all())
    assert bool(rms[3, 5].isnan()) and bool(layer[3].isnan().all())
    ref.check(rms[5:], *ref.norm(x[5:])[1])  # rows keep to themselves


def test_norm_empty_and_refused(ops):
    x = torch.zeros(0, 64, dtype=F16, device="cuda")
    assert ops.norm(x).shape == (0, 64)
    x = torch.zeros(4, 64, dtype=F16, device="cuda")
    for bad in (dict(weight=torch.zeros(63, dtype=F16, device="cuda")), dict(weight=torch.zeros(64, device="cuda")),
                dict(scale=torch.zeros(1, 64, dtype=F16, device="cuda"), group=2), dict(kind="batch"), dict(group=0),
                dict(out=torch.zeros(4, 63, dtype=F16, device="cuda")), dict(weight=torch.zeros(64, dtype=F16)),
                dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(InvalidArgument):
            ops.norm(x, **bad)
    with pytest.raises(InvalidArgument):
        ops.norm(x.double())
    with pytest.raises(InvalidArgument):
        ops.norm(x.t())
    with pytest.raises(InvalidArgument):
        ops.residual_norm(x, None)
    with pytest.raises(Unsupported):
        ops.norm(torch.zeros(2, 8193, dtype=F16, device="cuda"))


# ---------------------------------------------------------------------------------------- rotary


def series(pairs):
    f = [10000.0 ** (-i / n) for n in pairs for i in range(n)]
    return torch.tensor(f, dtype=torch.float64, device="cuda")


def places(gen, tokens, most=1800):
    return torch.randint(0, most, (tokens, 3), generator=gen, device="cuda").to(torch.int32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,pairs", [
    (1, 1, 2, (1, 0, 0)), (1, 16, 128, (16, 24, 24)), (5, 3, 64, (8, 12, 12)), (9, 2, 100, (3, 7, 5)), (700, 4, 128, (16, 22, 22)),
    (2401, 2, 64, (0, 8, 8)), (33, 5, 6, (1, 1, 1)), (17, 1, 512, (100, 80, 76)), (64, 2, 64, (0, 0, 0)), (40, 7, 72, (12, 12, 12))])
def test_rotary(ops, dtype, interleaved, tokens, heads, dim, pairs):
    g = generator(tokens + 31 * heads + dim)
    x, at, f = normal(g, (tokens, heads, dim), dtype), places(g, tokens), series(pairs)
    want, bound = ref.rotary(x, at, f, pairs, interleaved)
    out = ops.rotary(x, at, f, pairs, interleaved=interleaved)
    ref.check(out, want, bound)
    assert torch.equal(ops.rotary(x, at, f, pairs, interleaved=interleaved, out=x), out)  # in place


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,pairs", [
    (40007, 4, 64, (8, 12, 12)), (20001, 7, 80, (13, 13, 11)), (9000, 6, 128, (16, 22, 22)), (50001, 1, 128, (0, 31, 30)),
    (3001, 2, 512, (100, 80, 76))])
def test_rotary_of_many_tokens(ops, dtype, interleaved, tokens, heads, dim, pairs):
    """Enough rows for the kernel that copies them whole; also from and into strided rows, and in place."""
    g = generator(tokens + dim)
    wide = normal(g, (tokens, heads + 2, dim + 16), dtype)
    at, f = places(g, tokens), series(pairs)
    x = wide[:, 1:1 + heads, :dim]
    want, bound = ref.rotary(x, at, f, pairs, interleaved)
    out = ops.rotary(x, at, f, pairs, interleaved=interleaved)
    ref.check(out, want, bound)
    whole = x.contiguous()
    assert torch.equal(ops.rotary(whole, at, f, pairs, interleaved=interleaved), out)
    assert torch.equal(ops.rotary(whole, at, f, pairs, interleaved=interleaved, out=whole), out)
    before = wide.clone()
    assert ops.rotary(x, at, f, pairs, interleaved=interleaved, out=x) is x
    assert torch.equal(x, out)
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, -1], before[:, -1])
    assert torch.equal(wide[:, :, dim:], before[:, :, dim:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_strides_and_far_positions(ops, interleaved):
    g = generator(3)
    wide = normal(g, (50, 9, 144), BF16)
    at = places(g, 50, 2 ** 31 - 1)
    at[0] = torch.tensor([-(2 ** 31), -1, 2 ** 31 - 1])
    pairs = (16, 16, 16)
    for x in (wide[:, 2:6, 8:136], wide[:, 1:4, 1:129], wide.transpose(0, 1)[:, :, :128][:9, :50].transpose(0, 1)):
        want, bound = ref.rotary(x, at, series(pairs), pairs, interleaved)
        ref.check(ops.rotary(x, at, series(pairs), pairs, interleaved=interleaved), want, bound)


def test_rotary_refused(ops):
    x = torch.zeros(4, 2, 64, dtype=F16, device="cuda")
    at, f = torch.zeros(4, 3, dtype=torch.int32, device="cuda"), series((8, 8, 8))
    assert ops.rotary(x[:0], at[:0], f, (8, 8, 8)).shape == (0, 2, 64)
    for bad in (dict(positions=at.long()), dict(positions=at[:3]), dict(frequencies=f.float()), dict(pairs=(8, 8, 9)),
                dict(pairs=(8, 16)), dict(pairs=(-8, 16, 16)), dict(out=x[:, :1]), dict(x=x[0]), dict(x=x.double()),
                dict(x=x.transpose(1, 2))):
        with pytest.raises(InvalidArgument):
            ops.rotary(**(dict(x=x, positions=at, frequencies=f, pairs=(8, 8, 8)) | bad))


# ---------------------------------------------------------------------------------------- append


def paged(gen, lengths, steps, heads, dim, page, dtype, spare=2):
    """A cache of shuffled pages full of values, the streams' table (-1 where a stream has no page), starts, lengths."""
    need = [max(0, -(-n // page)) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen, device="cuda").int()
    table = torch.full((len(lengths), max(need + [1]) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([sum(steps[:i]) for i in range(len(steps) + 1)], dtype=torch.int32, device="cuda")
    k, v = normal(gen, (total, page, heads, dim), dtype), normal(gen, (total, page, heads, dim), dtype)
    return k, v, table, starts, torch.tensor(lengths, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lengths,steps,heads,q_heads,dim,page", [
    ([1], [1], 1, 1, 64, 16), ([5, 1, 40], [1, 1, 1], 4, 16, 128, 16), ([300, 7, 64], [64, 7, 0], 2, 6, 64, 48),
    ([33] * 70, [k % 4 for k in range(70)], 2, 2, 40, 1), ([1200, 900], [1200, 3], 3, 3, 128, 100)])
def test_append(ops, dtype, lengths, steps, heads, q_heads, dim, page):
    g = generator(sum(lengths) + dim)
    k_cache, v_cache, table, starts, have = paged(g, lengths, steps, heads, dim, page, dtype)
    tokens = sum(steps) + 3  # three tokens of padding that belong to no stream
    qkv = normal(g, (tokens, q_heads + 2 * heads, dim), dtype)
    q, k, v = qkv.split((q_heads, heads, heads), 1)
    pairs = (dim // 8, dim // 8, dim // 8)
    at, f = places(g, tokens), series(pairs)
    turned, bound = ref.rotary(qkv, at, f, pairs, False)
    # exact for a copied value; a rotated key is the one the rotary operator gives
    want_k, want_v = k_cache.clone(), v_cache.clone()
    ref.append(ops.rotary(k, at, f, pairs), v, want_k, want_v, table, starts, have)
    out = ops.append(k, v, k_cache, v_cache, table, starts, have, q=q, positions=at, frequencies=f, pairs=pairs)
    assert torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)
    ref.check(out, turned[:, :q_heads], bound[:, :q_heads])
    # without a rotation and without queries
    ref.append(k, v, want_k, want_v, table, starts, have)
    assert ops.append(k, v, k_cache, v_cache, table, starts, have) is None
    assert torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,q_heads,dim,page,pairs", [(4, 8, 128, 64, (16, 24, 24)), (3, 9, 72, 20, (7, 11, 5)),
                                                          (2, 0, 64, 16, (8, 12, 12))])
def test_append_of_many_tokens(ops, dtype, heads, q_heads, dim, page, pairs):
    """Enough rows for the kernel that copies them whole, into a cache with heads before slots as well; a
    stream without a step, one that has no pages, and padding."""
    g = generator(dim)
    lengths, steps = [9000, 4000, 12345, 77, 5000], [9000, 0, 12000, 77, 4999]
    k_cache, v_cache, table, starts, have = paged(g, lengths, steps, heads, dim, page, dtype)
    table[3] = -1
    tokens = sum(steps) + 5
    qkv = normal(g, (tokens, q_heads + 2 * heads, dim), dtype)
    q, k, v = qkv.split((q_heads, heads, heads), 1)
    at, f = places(g, tokens), series(pairs)
    turned = ops.rotary(qkv, at, f, pairs)
    want_k, want_v = k_cache.clone(), v_cache.clone()
    stream = torch.repeat_interleave(torch.arange(5, device="cuda"), torch.tensor(steps, device="cuda"))
    token = torch.arange(sum(steps), device="cuda")
    position = have.long()[stream] - starts.long()[stream + 1] + token
    pages = table[stream, position // page].long()
    stored = pages >= 0
    want_k[pages[stored], (position % page)[stored]] = turned[token[stored], q_heads:q_heads + heads]
    want_v[pages[stored], (position % page)[stored]] = v[token[stored]]
    for k_to, v_to in ((k_cache.clone(), v_cache.clone()),
                       (k_cache.transpose(1, 2).contiguous().transpose(1, 2), v_cache.transpose(1, 2).contiguous().transpose(1, 2))):
        out = ops.append(k, v, k_to, v_to, table, starts, have, q=q if q_heads else None, positions=at, frequencies=f, pairs=pairs)
        assert torch.equal(k_to, want_k) and torch.equal(v_to, want_v)
        if q_heads:
            assert torch.equal(out, turned[:, :q_heads])
    assert ops.lib.dcn_device_error() == 0


def test_append_leaves_out_what_has_no_place(ops):
    """Negative positions, positions past the table and page ids outside the cache are not stored."""
    g = generator(11)
    k_cache, v_cache, table, starts, lengths = paged(g, [6, 40, 20, 33], [10, 4, 20, 33], 2, 64, 16, F16)
    table = table[:, :2].contiguous()  # stream 1 and 3 run past two pages
    table[2, 0] = 1 << 20
    table[2, 1] = -5
    k, v = normal(g, (67, 2, 64), F16), normal(g, (67, 2, 64), F16)
    want_k, want_v = k_cache.clone(), v_cache.clone()
    ref.append(k, v, want_k, want_v, table, starts, lengths)
    ops.append(k, v, k_cache, v_cache, table, starts, lengths)
    assert torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)


def test_append_strided_cache_past_32_bits(ops):
    """Keys and values of a page side by side, heads before slots, and pages past element 2^31."""
    g = generator(12)
    pages, page, heads, dim = 5100, 64, 16, 128
    both = torch.empty(pages, heads, 2, page, dim, dtype=F16, device="cuda")  # 2.7e9 elements
    k_cache, v_cache = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    table = torch.tensor([[5099, 0], [4999, 5098]], dtype=torch.int32, device="cuda")
    both[table.flatten().long()] = 0
    starts = torch.tensor([0, 70, 170], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([70, 120], dtype=torch.int32, device="cuda")
    k, v = normal(g, (170, heads, dim), F16), normal(g, (170, heads, dim), F16)
    ops.append(k, v, k_cache, v_cache, table, starts, lengths)
    for b, (lo, hi, n) in enumerate(((0, 70, 70), (70, 170, 120))):
        got_k, got_v = (c[table[b].long()].flatten(0, 1)[n - (hi - lo):n] for c in (k_cache, v_cache))
        assert torch.equal(got_k, k[lo:hi]) and torch.equal(got_v, v[lo:hi])
    assert not bool(both[table[0, 1].long()][:, :, 6:].any())


def test_append_refused_and_other_stream(ops):
    g = generator(13)
    k_cache, v_cache, table, starts, lengths = paged(g, [20, 30], [4, 5], 2, 64, 16, BF16)
    k, v = normal(g, (9, 2, 64), BF16), normal(g, (9, 2, 64), BF16)
    good = dict(k=k, v=v, k_cache=k_cache, v_cache=v_cache, table=table, starts=starts, lengths=lengths)
    for bad in (dict(k=k[:, :1]), dict(v=v.half()), dict(v_cache=v_cache[:, :8]), dict(table=table.long()), dict(starts=starts[:2]),
                dict(lengths=lengths.long()), dict(table=table[0]), dict(q=k[..., :32]), dict(q_out=k), dict(pairs=(1, 1, 1)),
                dict(k=k.cpu()), dict(k_cache=k_cache.transpose(2, 3))):
        with pytest.raises(InvalidArgument):
            ops.append(**(good | bad))
    want_k, want_v = k_cache.clone(), v_cache.clone()
    ref.append(k, v, want_k, want_v, table, starts, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = ops.append(**good, q=k, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, k) and torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,width,group,post", [(4101, 1024, 16, False), (4101, 1024, 17, True), (20011, 256, 130, True),
                                                   (50003, 96, 400, False), (8200, 520, 100000, False), (9001, 1024, 5, False)])
def test_residual_norm_by_rows_and_groups(ops, dtype, rows, width, group, post):
    """On both sides of the sizes from which a block folds its groups' vectors; its share of rows is no multiple
    of its warps, and ends inside a group."""
    g = generator(rows + group)
    groups = -(-rows // group)
    x, residual = normal(g, (rows, width), dtype, 2.0) - 0.5, normal(g, (rows, width), dtype, 3.0)
    shift, scale, gate = normal(g, (groups, 3, width), dtype, 0.4).unbind(1)
    args = dict(gate=gate, kind="layer", weight=1 + normal(g, (width,), dtype, 0.1), scale=scale, shift=shift, group=group)
    if post:
        args |= dict(post_weight=1 + normal(g, (width,), dtype, 0.1), post_bias=normal(g, (width,), dtype, 0.1))
    hidden, out = ops.residual_norm(x, residual, **args)
    want_hidden, want_out = ref.norm(x, residual, **args)
    ref.check(hidden, *want_hidden)
    ref.check(out, *want_out)
    plain = dict(scale=scale, shift=shift, group=group)
    ref.check(ops.norm(x, **plain), *ref.norm(x, **plain)[1])


@pytest.mark.parametrize("group", [0, -1, 2**63, 2**64 + 1])
def test_norm_group_out_of_range(ops, group):
    """Refused, not cut to its low bits."""
    with pytest.raises(InvalidArgument):
        ops.norm(torch.zeros(2, 64, dtype=F16, device="cuda"), group=group)
