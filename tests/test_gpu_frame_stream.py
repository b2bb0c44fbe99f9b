"""GPU: the streaming block of examples/frame_stream.py against the same block in FP64 without a cache."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "frame_stream.py"
    spec = importlib.util.spec_from_file_location("frame_stream", path)
    module = importlib.util.module_from_spec(spec)
    import sys

    sys.modules["frame_stream"] = module
    spec.loader.exec_module(module)
    return module


def test_block_follows_streams_past_its_window(example):
    """Seven frames with a window of three and one sink: pages are used again, early frames leave.

    Bound: FP16 roundings at eight places of a frame (two norms, four products, weights, result), each
    2^-11 relative and independent, grow by the block's products and norms by less than four:
    sqrt(8) * 2^-11 * 4 = 6e-3 of the result's 2-norm."""
    streams, frames, window, sinks = 3, 7, 3, 1
    w = example.Weights.random(streams, seed=3)
    block = example.FrameStream(w, streams, window=window, sinks=sinks)
    g = torch.Generator(device="cuda").manual_seed(5)
    tokens, heads, kv, dim = example.TOKENS, example.HEADS, example.KV_HEADS, example.HEAD_DIM
    keys, values = [], []
    shift1, scale1, gate1, shift2, scale2, gate2 = w.modulation.unbind(1)
    for f in range(frames):
        x = torch.randn(streams * tokens, example.WIDTH, generator=g, device="cuda").half()
        got = block.step(x)
        y = ref.norm(x, kind="layer", weight=w.norm1, scale=scale1, shift=shift1, group=tokens)[1][0]
        qkv = (y @ w.qkv.double()).view(-1, heads + 2 * kv, dim)
        qk = ref.rotary(qkv[:, :heads + kv].float(), block.positions, block.frequencies, example.PAIRS, False)[0]
        keys.append(qk[:, heads:].view(streams, tokens, kv, dim))
        values.append(qkv[:, heads + kv:].view(streams, tokens, kv, dim))
        seen = [i for i in range(f + 1) if i < sinks or i > f - window]
        k = torch.cat([keys[i] for i in seen], 1).repeat_interleave(heads // kv, 2)
        v = torch.cat([values[i] for i in seen], 1).repeat_interleave(heads // kv, 2)
        q = qk[:, :heads].view(streams, tokens, heads, dim)
        p = torch.softmax(torch.einsum("sqhd,skhd->shqk", q, k) * dim ** -0.5, -1)
        attended = torch.einsum("shqk,skhd->sqhd", p, v).reshape(-1, heads * dim) @ w.out.double()
        group = torch.arange(streams * tokens, device="cuda") // tokens
        hidden = x.double() + gate1.double()[group] * attended
        n = ref.normalised(hidden, "layer", 1e-6)[0] * w.norm2.double()
        n = n * (1 + scale2.double()[group]) + shift2.double()[group]
        m = torch.nn.functional.silu(n @ w.up.double()) @ w.down.double()
        want = hidden + gate2.double()[group] * m
        off = ((got.double() - want).norm() / want.norm()).item()
        assert off <= 6e-3, (f, off)
    assert block.ops.lib.dcn_device_error() == 0


def test_example_runs_behind_the_convolution(example, monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["frame_stream.py", "--streams", "2", "--frames", "3"])
    example.main()
    assert "finite: True" in capsys.readouterr().out


def test_stream_runs_on_for_good(example):
    """Past 1,024 frames of one stream, where a table with a column a frame would have to end.  Bound: as above."""
    window, sinks, last = 2, 1, 1030
    w = example.Weights.random(1, seed=4)
    block = example.FrameStream(w, 1, window=window, sinks=sinks)
    g = torch.Generator(device="cuda").manual_seed(6)
    tokens, heads, kv, dim = example.TOKENS, example.HEADS, example.KV_HEADS, example.HEAD_DIM
    shift1, scale1, gate1, shift2, scale2, gate2 = (m.double() for m in w.modulation.unbind(1))
    frames = torch.randn(16, tokens, example.WIDTH, generator=g, device="cuda").half()
    keys, values = {}, {}
    for f in range(last):
        x = frames[f % 16]
        got = block.step(x)
        if sinks <= f < 1020:
            continue
        y = ref.normalised(x.double(), "layer", 1e-6)[0] * w.norm1.double() * (1 + scale1) + shift1
        qkv = (y @ w.qkv.double()).view(-1, heads + 2 * kv, dim)
        positions = block.positions.clone()
        positions[:, 0] = f
        qk = ref.rotary(qkv[:, :heads + kv].float(), positions, block.frequencies, example.PAIRS, False)[0]
        keys[f], values[f] = qk[:, heads:], qkv[:, heads + kv:]
        if f < 1022:
            continue
        seen = [i for i in keys if i < sinks or i > f - window]
        k = torch.cat([keys[i] for i in seen]).repeat_interleave(heads // kv, 1)
        v = torch.cat([values[i] for i in seen]).repeat_interleave(heads // kv, 1)
        p = torch.softmax(torch.einsum("qhd,khd->hqk", qk[:, :heads], k) * dim ** -0.5, -1)
        attended = torch.einsum("hqk,khd->qhd", p, v).reshape(-1, heads * dim) @ w.out.double()
        hidden = x.double() + gate1 * attended
        n = ref.normalised(hidden, "layer", 1e-6)[0] * w.norm2.double() * (1 + scale2) + shift2
        want = hidden + gate2 * (torch.nn.functional.silu(n @ w.up.double()) @ w.down.double())
        off = ((got.double() - want).norm() / want.norm()).item()
        assert off <= 6e-3, (f, off)
    assert block.ops.lib.dcn_device_error() == 0
