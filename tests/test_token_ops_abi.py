"""The token operators' refusals, without a GPU: an invalid call stops at its own status before the
device is touched, and a valid one gets as far as DCN_ERR_NO_DEVICE."""

from __future__ import annotations

import ctypes

import pytest

from jasnamacos_b200 import _native

OK, SHAPE, NO_DEVICE = _native.DCN_OK, _native.DCN_ERR_INVALID_SHAPE, _native.DCN_ERR_NO_DEVICE
ARGUMENT, UNSUPPORTED = _native.DCN_ERR_INVALID_ARGUMENT, _native.DCN_ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def lib():
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-device status")
    return _native.load()


def heads(data=256, token=64, head=64):
    return _native.DcnHeads(data, token, head)


def rotation(pairs=(4, 6, 6), frequencies=256, positions=256, interleaved=0):
    return _native.DcnRotation(frequencies, positions, pairs, interleaved)


def cache(**changes):
    fields = dict(keys=256, values=256, key_page_stride=1024, key_slot_stride=64, key_head_stride=64,
                  value_page_stride=1024, value_slot_stride=64, value_head_stride=64, pages=4, page_size=16, heads=1,
                  head_dim=64, dtype=_native.DCN_DTYPE_F16, streams=2, table_columns=2, reserved=0, table_stride=2,
                  table=256, starts=256, lengths=256)
    fields.update(changes)
    return _native.DcnPagedCache(**fields)


def attention_args(**changes):
    fields = dict(tokens=8, q_heads=2, max_q=4, max_kv=32, window=4, sinks=1, frame=1, scale=0.125, reserved=0)
    fields.update(changes)
    return _native.DcnTokenAttentionArgs(**fields)


def norm_args(**changes):
    fields = dict(rows=4, group=1, width=64, dtype=_native.DCN_DTYPE_F16, kind=0, post=0, epsilon=1e-6, residual_scale=1.0,
                  x=256, residual=256, weight=256, hidden=256, out=256, x_stride=64, residual_stride=64, hidden_stride=64,
                  out_stride=64)
    fields.update(changes)
    return _native.DcnTokenNormArgs(**fields)


def test_struct_sizes_match_the_header(tmp_path):
    """The ctypes mirrors have the C structs' sizes and last offsets."""
    import shutil
    import subprocess
    from pathlib import Path

    include = Path(__file__).resolve().parent.parent / "include"
    mirrors = {"dcn_heads": _native.DcnHeads, "dcn_rotation": _native.DcnRotation, "dcn_paged_cache": _native.DcnPagedCache,
               "dcn_token_attention_args": _native.DcnTokenAttentionArgs, "dcn_token_norm_args": _native.DcnTokenNormArgs}
    lines = []
    for name, mirror in mirrors.items():
        fields = [f[0] for f in mirror._fields_]
        lines.append(f'printf("%zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f}));' for f in fields]
        lines.append('printf("\\n");')
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "dcn_b200.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run([shutil.which("gcc"), "-std=c11", f"-I{include}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    for line, mirror in zip(out, mirrors.values()):
        want = [ctypes.sizeof(mirror)] + [getattr(mirror, f[0]).offset for f in mirror._fields_]
        assert [int(v) for v in line.split()] == want, mirror.__name__


@pytest.mark.parametrize("dtype,tokens,n,dim,rot,x,want", [
    (1, 8, 2, 64, rotation(), heads(), NO_DEVICE),
    (0, 8, 2, 64, rotation((0, 0, 0), None, None), heads(), NO_DEVICE),
    (2, 0, 2, 64, None, None, OK),                        # no tokens: nothing to do
    (3, 8, 2, 64, rotation(), heads(), ARGUMENT),         # unknown type
    (1, -1, 2, 64, rotation(), heads(), SHAPE),
    (1, 8, 0, 64, rotation(), heads(), SHAPE),
    (1, 8, 2, 63, rotation(), heads(), SHAPE),            # odd head_dim
    (1, 8, 2, 514, rotation(), heads(), UNSUPPORTED),
    (1, 8, 2, 30, rotation(), heads(), SHAPE),            # more pairs than the head has
    (1, 8, 2, 64, rotation((-1, 4, 4)), heads(), SHAPE),
    (1, 8, 2, 64, rotation(interleaved=2), heads(), ARGUMENT),
    (1, 8, 2, 64, rotation(frequencies=None), heads(), ARGUMENT),
    (1, 8, 2, 64, rotation(frequencies=260), heads(), ARGUMENT),
    (1, 8, 2, 64, rotation(positions=None), heads(), ARGUMENT),
    (1, 8, 2, 64, None, heads(), ARGUMENT),
    (1, 8, 2, 64, rotation(), None, ARGUMENT),
    (1, 8, 2, 64, rotation(), heads(data=257), ARGUMENT),
    (1, 8, 2, 64, rotation(), heads(token=-64), ARGUMENT),
])
def test_rotary_refusals(lib, dtype, tokens, n, dim, rot, x, want):
    assert lib.dcn_token_rotary(dtype, tokens, n, dim, rot, x, heads(), None) == want
    assert lib.dcn_token_rotary(dtype, tokens, n, dim, rot, heads() if x else None, x, None) == want


@pytest.mark.parametrize("changes,want", [
    ({}, NO_DEVICE), (dict(streams=0, lengths=None, table=None), NO_DEVICE), (dict(table_columns=0, table=None), NO_DEVICE),
    (dict(pages=0), SHAPE), (dict(page_size=0), SHAPE), (dict(heads=0), SHAPE), (dict(head_dim=0), SHAPE),
    (dict(streams=-1), SHAPE), (dict(table_columns=-1), SHAPE), (dict(dtype=7), ARGUMENT), (dict(reserved=1), ARGUMENT),
    (dict(keys=None), ARGUMENT), (dict(values=257), ARGUMENT), (dict(key_page_stride=-1), ARGUMENT),
    (dict(value_slot_stride=1 << 40), ARGUMENT), (dict(starts=None), ARGUMENT), (dict(lengths=None), ARGUMENT),
    (dict(table=None), ARGUMENT), (dict(table=258), ARGUMENT), (dict(head_dim=514), UNSUPPORTED),
])
def test_append_refusals(lib, changes, want):
    c = cache(**changes)
    assert lib.dcn_token_append(c, 8, None, heads(), heads(), 2, heads(), heads(), None) == want


def test_append_tensor_refusals(lib):
    c = cache()
    assert lib.dcn_token_append(c, 8, None, heads(), heads(), 0, None, None, None) == NO_DEVICE
    assert lib.dcn_token_append(c, 0, None, None, None, 0, None, None, None) == OK
    assert lib.dcn_token_append(c, 8, None, None, heads(), 0, None, None, None) == ARGUMENT
    assert lib.dcn_token_append(c, 8, None, heads(), heads(data=257), 0, None, None, None) == ARGUMENT
    assert lib.dcn_token_append(c, 8, None, heads(), heads(), 2, heads(), None, None) == ARGUMENT
    assert lib.dcn_token_append(c, 8, None, heads(), heads(), -1, None, None, None) == SHAPE
    assert lib.dcn_token_append(c, -1, None, heads(), heads(), 0, None, None, None) == SHAPE
    assert lib.dcn_token_append(c, 8, rotation((20, 20, 20)), heads(), heads(), 0, None, None, None) == SHAPE
    assert lib.dcn_token_append(None, 8, None, heads(), heads(), 0, None, None, None) == ARGUMENT


@pytest.mark.parametrize("changes,want", [
    ({}, NO_DEVICE), (dict(tokens=0), OK), (dict(tokens=-1), SHAPE), (dict(q_heads=0), SHAPE), (dict(max_q=-1), SHAPE),
    (dict(max_kv=-1), SHAPE), (dict(tokens=1 << 31), SHAPE), (dict(window=0), ARGUMENT), (dict(sinks=-1), ARGUMENT),
    (dict(frame=0), ARGUMENT), (dict(scale=float("nan")), ARGUMENT), (dict(reserved=1), ARGUMENT),
])
def test_attention_refusals(lib, changes, want):
    buffer = ctypes.c_void_p(1 << 20)
    assert lib.dcn_token_attention(cache(), attention_args(**changes), heads(), heads(), buffer, 1 << 40, None) == want


def test_attention_tensor_refusals(lib):
    a = attention_args()
    ws = ctypes.c_void_p(1 << 20)
    call = lambda c, q, o, args=a: lib.dcn_token_attention(c, args, q, o, ws, 1 << 40, None)  # noqa: E731
    assert call(cache(), None, heads()) == ARGUMENT
    assert call(cache(), heads(), heads(data=257)) == ARGUMENT
    assert call(cache(heads=3, key_head_stride=8, value_head_stride=8), heads(), heads()) == SHAPE  # 2 query heads, 3 key heads
    assert call(cache(head_dim=258), heads(), heads()) == UNSUPPORTED
    assert call(cache(streams=0, lengths=None, table=None), heads(), heads()) == OK
    assert call(cache(), heads(), heads(), None) == ARGUMENT


@pytest.mark.parametrize("changes,want", [
    ({}, NO_DEVICE), (dict(rows=0, x=None), OK), (dict(residual=None, hidden=None), NO_DEVICE), (dict(out=None), NO_DEVICE),
    (dict(rows=-1), SHAPE), (dict(width=0), SHAPE), (dict(group=0), SHAPE), (dict(width=8193), UNSUPPORTED),
    (dict(kind=2), ARGUMENT), (dict(post=2), ARGUMENT), (dict(dtype=3), ARGUMENT), (dict(epsilon=-1.0), ARGUMENT),
    (dict(epsilon=float("nan")), ARGUMENT), (dict(x=None), ARGUMENT), (dict(hidden=None, out=None), ARGUMENT),
    (dict(residual=None), ARGUMENT), (dict(residual=None, hidden=None, gate=256), ARGUMENT),
    (dict(residual=None, hidden=None, post=1), ARGUMENT), (dict(post_weight=256), ARGUMENT), (dict(weight=257), ARGUMENT),
    (dict(x_stride=-1), ARGUMENT), (dict(shift=256, shift_stride=1 << 40), ARGUMENT),
])
def test_norm_refusals(lib, changes, want):
    assert lib.dcn_token_norm(norm_args(**changes), None) == want


@pytest.mark.parametrize("tokens", [1 << 31, 1 << 61, (1 << 63) - 1])
def test_attention_token_counts_past_32_bits(lib, tokens):
    """Refused as such: tokens * q_heads does not wrap to something small."""
    args = attention_args(tokens=tokens, q_heads=8)
    assert lib.dcn_token_attention_workspace_bytes(cache(), args) == 0
    assert lib.dcn_token_attention(cache(), args, heads(), heads(), None, 0, None) == SHAPE


@pytest.mark.parametrize("q_heads", [2, 8])
def test_attention_workspace_with_loose_limits(lib, q_heads):
    """max_q and max_kv far past the tokens and the table cost no more scratch than the tight ones."""
    wide = cache(table_columns=1024, table_stride=1024)
    tight = lib.dcn_token_attention_workspace_bytes(wide, attention_args(q_heads=q_heads, max_q=8, max_kv=16384, window=1 << 30))
    loose = lib.dcn_token_attention_workspace_bytes(
        wide, attention_args(q_heads=q_heads, max_q=2**31 - 1, max_kv=2**31 - 1, window=1 << 30))
    assert 0 < tight == loose
