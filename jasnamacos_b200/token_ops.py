"""Token operators: a streaming transformer block next to the deformable convolution.

Tokens are patches of a tile's features, frame after frame.  A block over them is library matrix
products plus the four operators here (``dcn_token_*`` of ``include/dcn_b200.h``):

* :meth:`CudaTokenOps.norm`, :meth:`CudaTokenOps.residual_norm` -- the norms before and after a block,
  with its gate, residual scale and modulation
* :meth:`CudaTokenOps.rotary` -- rotary positions over (time, row, column)
* :meth:`CudaTokenOps.append` -- a step's keys and values into a paged cache, rotated on the way,
  and its queries rotated with them
* :meth:`CudaTokenOps.attention` -- the step's queries over the cache: the last ``window`` frames and
  the first ``sinks`` frames

The reference has no counterpart: its network carries information between frames by flow and
convolution only.  Everything computes in ``libdcn_b200.so``; PyTorch provides device memory and
streams.  There is no CPU fallback.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _native
from .deform_conv import DeviceUnavailable, InvalidArgument, raise_for_status

_DTYPES = {torch.float32: _native.DCN_DTYPE_F32, torch.float16: _native.DCN_DTYPE_F16,
           torch.bfloat16: _native.DCN_DTYPE_BF16}
_KINDS = {"rms": _native.DCN_NORM_RMS, "layer": _native.DCN_NORM_LAYER}
# ctypes keeps an integer's low bits only: the heads and widths of a larger tensor go in as this, which the library
# refuses.
_MOST = (1 << 31) - 1


def _said(name, t, wanted) -> InvalidArgument:
    return InvalidArgument(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device} with strides {t.stride()}; {wanted} is wanted")


class CudaTokenOps:
    """The token operators on CUDA tensors.

    Methods enqueue on the current stream of the tensors' device, or on ``stream``, and return without
    waiting.  Token tensors are ``[tokens, heads, head_dim]`` with any strides but a unit one along
    ``head_dim``; results are new tensors unless ``out`` is given.
    """

    def __init__(self, device: int | None = None):
        self.lib = _native.load()
        if not torch.cuda.is_available():
            raise DeviceUnavailable()
        self.device = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        self._index = self.device.index

    # -- checks ------------------------------------------------------------------
    # Small calls take some microseconds on the GPU, so a call's own Python counts: each check is one
    # comparison of plain values, and messages are only made where one fails.
    def _dtype(self, t) -> int:
        dtype = _DTYPES.get(t.dtype)
        if dtype is None:
            raise InvalidArgument(f"element type {t.dtype}: float32, float16 or bfloat16 is wanted")
        return dtype

    def _tokens(self, name, t, shape, dtype) -> _native.DcnHeads:
        """A [tokens][heads][head_dim] tensor with unit stride along head_dim on this device."""
        if t.shape != shape or t.dtype != dtype or t.get_device() != self._index:
            raise _said(name, t, f"{tuple(shape)} {dtype} on {self.device}")
        token, head, unit = t.stride()
        if unit != 1 and shape[2] > 1:
            raise _said(name, t, "unit stride along the last dimension")
        return _native.DcnHeads(t.data_ptr(), token, head)

    def _whole(self, name, t, shape, dtype) -> int:
        """The address of a contiguous tensor of a given shape and type on this device."""
        if t.shape != shape or t.dtype != dtype or t.get_device() != self._index or not t.is_contiguous():
            raise _said(name, t, f"a contiguous {tuple(shape)} {dtype} tensor on {self.device}")
        return t.data_ptr()

    def _call(self, stream, function, *args) -> None:
        """Calls the library on this operator's device and the given or current stream."""
        index = self._index
        handle = torch._C._cuda_getCurrentRawStream(index) if stream is None else stream.cuda_stream
        if torch._C._cuda_getDevice() == index:
            status = function(*args, handle or None)
        else:
            with torch.cuda.device(index):
                status = function(*args, handle or None)
        if status != _native.DCN_OK:
            raise_for_status(status, function.__name__)

    def _new(self, like, stream):
        """A contiguous tensor like another one, from the memory of the stream that will write it."""
        if stream is None:
            return torch.empty_like(like, memory_format=torch.contiguous_format)
        with torch.cuda.stream(stream):
            return torch.empty_like(like, memory_format=torch.contiguous_format)

    def _rotation(self, positions, frequencies, pairs, interleaved, tokens) -> _native.DcnRotation:
        if len(pairs) != 3 or min(pairs) < 0:
            raise InvalidArgument(f"pairs {pairs}: one count for each of three axes is wanted")
        time, row, column = pairs
        return _native.DcnRotation(self._whole("frequencies", frequencies, (time + row + column,), torch.float64),
                                   self._whole("positions", positions, (tokens, 3), torch.int32), (time, row, column),
                                   1 if interleaved else 0)

    def _cache(self, k_cache, v_cache, table, starts, lengths) -> _native.DcnPagedCache:
        shape = k_cache.shape
        if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype != k_cache.dtype:
            raise InvalidArgument(f"k_cache {tuple(shape)} {k_cache.dtype} and v_cache {tuple(v_cache.shape)} "
                                  f"{v_cache.dtype}: two [pages, page_size, heads, head_dim] tensors of one type are wanted")
        k_page, k_slot, k_head, k_unit = k_cache.stride()
        v_page, v_slot, v_head, v_unit = v_cache.stride()
        index = self._index
        if k_cache.get_device() != index or v_cache.get_device() != index or k_unit != 1 or v_unit != 1:
            raise InvalidArgument(f"k_cache and v_cache need unit stride along head_dim and to be on {self.device}")
        if table.dim() != 2 or table.dtype != torch.int32 or table.get_device() != index:
            raise _said("table", table, f"a [streams, columns] int32 tensor on {self.device}")
        pages, page_size, heads, head_dim = shape
        streams, columns = table.shape
        if (pages | page_size | heads | head_dim | streams | columns) > _MOST:
            raise InvalidArgument(f"k_cache {tuple(shape)}, table {tuple(table.shape)}: 32-bit sizes are wanted")
        table_stride, unit = table.stride()
        if unit != 1 and columns > 1:
            raise _said("table", table, "unit stride along its rows")
        return _native.DcnPagedCache(
            k_cache.data_ptr(), v_cache.data_ptr(), k_page, k_slot, k_head, v_page, v_slot, v_head, pages, page_size, heads,
            head_dim, self._dtype(k_cache), streams, columns, 0, table_stride, table.data_ptr(),
            self._whole("starts", starts, (streams + 1,), torch.int32), self._whole("lengths", lengths, (streams,), torch.int32))

    # -- positions and cache -----------------------------------------------------
    def rotary(self, x, positions, frequencies, pairs, interleaved=False, out=None, stream=None):
        """Rotates the heads of `x` [tokens, heads, head_dim] by their token's position.

        Pair j belongs to axis 0 (time) for j < pairs[0], then to axis 1 (row) for pairs[1] pairs and to
        axis 2 (column) for pairs[2]; it turns by ``positions[token, axis] * frequencies[j]`` radians.
        `positions` is int32 [tokens, 3], `frequencies` float64 [sum(pairs)].  Pairs are elements
        (2j, 2j+1) when `interleaved`, else (j, j + sum(pairs)); elements past them stay.  `out` may be `x`."""
        if x.dim() != 3:
            raise InvalidArgument(f"x is {tuple(x.shape)}; [tokens, heads, head_dim] is wanted")
        shape = x.shape
        tokens, heads, head_dim = shape
        if heads > _MOST or head_dim > _MOST:
            heads = head_dim = _MOST
        x_at = self._tokens("x", x, shape, x.dtype)
        rotation = self._rotation(positions, frequencies, pairs, interleaved, tokens)
        if out is None:
            out = self._new(x, stream)
        out_at = self._tokens("out", out, shape, x.dtype)
        self._call(stream, self.lib.dcn_token_rotary, self._dtype(x), tokens, heads, head_dim, rotation, x_at, out_at)
        return out

    def append(self, k, v, k_cache, v_cache, table, starts, lengths, q=None, positions=None, frequencies=None,
               pairs=(0, 0, 0), interleaved=False, q_out=None, stream=None):
        """Writes a step's keys and values into the cache and rotates its queries, in one launch.

        `k`, `v` [tokens, kv_heads, head_dim]; stream b's tokens are [starts[b], starts[b+1]) and end at
        position lengths[b] - 1 (lengths count this step).  Position p lies in page table[b, p // page_size]
        of `k_cache`, `v_cache` [pages, page_size, kv_heads, head_dim].  With `positions`, keys and the
        queries `q` [tokens, q_heads, head_dim] are rotated as :meth:`rotary` does.  Returns the rotated
        queries (`q_out`, which may be `q`), or None without `q`."""
        cache = self._cache(k_cache, v_cache, table, starts, lengths)
        if k.dim() != 3:
            raise InvalidArgument(f"k is {tuple(k.shape)}; [tokens, kv_heads, head_dim] is wanted")
        tokens, dtype = k.shape[0], k_cache.dtype
        _, _, heads, head_dim = k_cache.shape
        k_at = self._tokens("k", k, (tokens, heads, head_dim), dtype)
        v_at = self._tokens("v", v, (tokens, heads, head_dim), dtype)
        rotation = None
        if positions is not None:
            rotation = self._rotation(positions, frequencies, pairs, interleaved, tokens)
        elif frequencies is not None or any(pairs):
            raise InvalidArgument("a rotation needs positions")
        q_heads, q_at, q_out_at = 0, None, None
        if q is not None:
            if q.dim() != 3:
                raise InvalidArgument(f"q is {tuple(q.shape)}; [tokens, q_heads, head_dim] is wanted")
            q_heads = q.shape[1]
            q_shape = (tokens, q_heads, head_dim)
            q_at = self._tokens("q", q, q_shape, dtype)
            if q_out is None:
                q_out = self._new(q, stream)
            q_out_at = self._tokens("q_out", q_out, q_shape, dtype)
        elif q_out is not None:
            raise InvalidArgument("q_out needs q")
        self._call(stream, self.lib.dcn_token_append, cache, tokens, rotation, k_at, v_at,
                   q_heads if q_heads <= _MOST else _MOST, q_at, q_out_at)
        return q_out

    # -- attention ---------------------------------------------------------------
    def _attention_args(self, tokens, q_heads, max_q, max_kv, window, sinks, frame, scale):
        if not 0 <= (max_q | max_kv | window | sinks | frame) <= _MOST:
            raise InvalidArgument(f"max_q {max_q}, max_kv {max_kv}, window {window}, sinks {sinks}, frame {frame}: "
                                  "32-bit counts are wanted")
        return _native.DcnTokenAttentionArgs(tokens, q_heads if q_heads <= _MOST else _MOST, max_q, max_kv, window, sinks, frame,
                                             scale, 0)

    def attention(self, q, k_cache, v_cache, table, starts, lengths, max_q, max_kv, window, sinks=0, frame=1, scale=None,
                  out=None, workspace=None, stream=None):
        """Attention of a step's queries `q` [tokens, q_heads, head_dim] over the cache of :meth:`append`.

        A frame is `frame` consecutive positions.  A query sees its own frame and those before it in the
        stream, of these the last `window` frames and the first `sinks` frames; frame = 1 is plain causal
        attention with a sliding window and first tokens that stay.  `max_q` bounds the streams' steps and
        `max_kv` their lengths.  `scale` defaults to head_dim ** -0.5.  A query that sees no key gives zeros;
        rows of tokens that belong to no stream are not written (nor cleared in a new `out`).  `workspace` (uint8, :meth:`attention_workspace_bytes`) is taken from PyTorch when not given."""
        if q.dim() != 3:
            raise InvalidArgument(f"q is {tuple(q.shape)}; [tokens, q_heads, head_dim] is wanted")
        cache = self._cache(k_cache, v_cache, table, starts, lengths)
        shape = q.shape
        tokens, q_heads, head_dim = shape
        q_at = self._tokens("q", q, (tokens, q_heads, cache.head_dim), k_cache.dtype)
        args = self._attention_args(tokens, q_heads, max_q, max_kv, window, sinks, frame,
                                    1.0 / math.sqrt(head_dim) if scale is None else scale)
        if out is None:
            out = self._new(q, stream)
        out_at = self._tokens("out", out, shape, q.dtype)
        need = self.lib.dcn_token_attention_workspace_bytes(cache, args)
        given, address = need, None
        if workspace is not None:
            if workspace.get_device() != self._index or not workspace.is_contiguous():
                raise _said("workspace", workspace, f"contiguous memory on {self.device}")
            given, address = workspace.numel() * workspace.element_size(), workspace.data_ptr()
        elif need:
            if stream is None:
                workspace = q.new_empty(need, dtype=torch.uint8)
            else:
                with torch.cuda.stream(stream):
                    workspace = q.new_empty(need, dtype=torch.uint8)
            address = workspace.data_ptr()
        self._call(stream, self.lib.dcn_token_attention, cache, args, q_at, out_at, address, given)
        return out

    def attention_workspace_bytes(self, q, k_cache, v_cache, table, starts, lengths, max_q, max_kv, window, sinks=0,
                                  frame=1) -> int:
        """Bytes of scratch that :meth:`attention` takes for these tensors."""
        cache = self._cache(k_cache, v_cache, table, starts, lengths)
        args = self._attention_args(q.shape[0], q.shape[1], max_q, max_kv, window, sinks, frame, 1.0)
        return int(self.lib.dcn_token_attention_workspace_bytes(cache, args))

    # -- norms -------------------------------------------------------------------
    def _vector(self, name, t, width, dtype):
        return None if t is None else self._whole(name, t, (width,), dtype)

    def _modulation(self, name, t, groups, width, dtype):
        """Address and row stride of a [groups, width] tensor with unit stride along its rows."""
        if t is None:
            return None, 0
        shape = t.shape
        if len(shape) != 2 or shape[1] != width or shape[0] < groups or t.dtype != dtype or t.get_device() != self._index:
            raise _said(name, t, f"[{groups}, {width}] {dtype} on {self.device}")
        row, unit = t.stride()
        if unit != 1 and width > 1:
            raise _said(name, t, "unit stride along its rows")
        return t.data_ptr(), row

    def _rows(self, name, t, shape, dtype):
        """Address and row stride of a [rows, width] tensor with unit stride along its rows."""
        if t is None:
            return None, 0
        if t.shape != shape or t.dtype != dtype or t.get_device() != self._index:
            raise _said(name, t, f"{tuple(shape)} {dtype} on {self.device}")
        row, unit = t.stride()
        if unit != 1 and shape[1] > 1:
            raise _said(name, t, "unit stride along its rows")
        return t.data_ptr(), row

    def _norm(self, x, residual, post, post_weight, post_bias, gate, residual_scale, kind, weight, bias, scale, shift, group,
              eps, hidden, out, stream):
        if x.dim() != 2:
            raise InvalidArgument(f"x is {tuple(x.shape)}; [rows, width] is wanted")
        shape, dtype = x.shape, x.dtype
        rows, width = shape
        if kind not in _KINDS:
            raise InvalidArgument(f"kind {kind!r}: 'rms' or 'layer' is wanted")
        if group is None:
            group = max(1, rows)
        if not 1 <= group < 1 << 63:
            raise InvalidArgument(f"group {group}: at least one row shares a modulation row")
        groups = -(-rows // group)
        x_at, x_stride = self._rows("x", x, shape, dtype)
        residual_at, residual_stride = self._rows("residual", residual, shape, dtype)
        hidden_at, hidden_stride = self._rows("hidden", hidden, shape, dtype)
        out_at, out_stride = self._rows("out", out, shape, dtype)
        gate_at, gate_stride = self._modulation("gate", gate, groups, width, dtype)
        scale_at, scale_stride = self._modulation("scale", scale, groups, width, dtype)
        shift_at, shift_stride = self._modulation("shift", shift, groups, width, dtype)
        args = _native.DcnTokenNormArgs(
            rows, group, width if width <= _MOST else _MOST, self._dtype(x), _KINDS[kind], post, eps, residual_scale, x_at, residual_at,
            self._vector("post_weight", post_weight, width, dtype), self._vector("post_bias", post_bias, width, dtype),
            self._vector("weight", weight, width, dtype), self._vector("bias", bias, width, dtype), gate_at, scale_at, shift_at,
            hidden_at, out_at, x_stride, residual_stride, hidden_stride, out_stride, gate_stride, scale_stride, shift_stride)
        self._call(stream, self.lib.dcn_token_norm, args)

    def norm(self, x, kind="rms", weight=None, bias=None, scale=None, shift=None, group=None, eps=1e-6, out=None, stream=None):
        """The norm before a block: ``(N(x) * weight + bias) * (1 + scale[g]) + shift[g]`` for the rows of
        `x` [rows, width], g = row // group (`group` None: one modulation row for all).  `kind` "rms" or
        "layer"; `scale`, `shift` [groups, width], rows of any stride; `out` may be `x`."""
        if out is None:
            out = self._new(x, stream)
        self._norm(x, None, 0, None, None, None, 1.0, kind, weight, bias, scale, shift, group, eps, None, out, stream)
        return out

    def residual_norm(self, x, residual, gate=None, post_weight=None, post_bias=None, residual_scale=1.0, kind="rms",
                      weight=None, bias=None, scale=None, shift=None, group=None, eps=1e-6, hidden=None, out=None, stream=None):
        """A block's end and the next one's norm, in one pass over the rows:

        ``hidden = residual_scale * residual + gate[g] * branch`` and
        ``out = (N(hidden) * weight + bias) * (1 + scale[g]) + shift[g]``,

        with branch = `x`, or ``N(x) * post_weight + post_bias`` when `post_weight` is given (the norm after
        the block).  Returns (hidden, out); `hidden` may be `residual` or `x`, `out` may be `x`."""
        if residual is None:
            raise InvalidArgument("residual_norm needs a residual")
        if post_bias is not None and post_weight is None:
            raise InvalidArgument("post_bias needs post_weight")
        if hidden is None:
            hidden = self._new(x, stream)
        if out is None:
            out = self._new(x, stream)
        self._norm(x, residual, int(post_weight is not None), post_weight, post_bias, gate, residual_scale, kind, weight, bias,
                   scale, shift, group, eps, hidden, out, stream)
        return hidden, out
