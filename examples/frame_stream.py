"""A transformer block that follows tile streams frame by frame, on the deformable convolution's features.

Per frame and stream: the DCN aligns the tile's features (64 channels, 64x64), they are cut into
4x4 patches (256 tokens of 1,024 values), and a block attends from them to the last `window` frames
and the first `sinks` frames of the stream.  The frames live in a paged cache, one frame a page; pages
of frames that left the window are used again, and so are their positions, so a stream may run on for
good (its time positions are 32-bit: two years at 30 frames a second).

    python examples/frame_stream.py --streams 8 --frames 30

Weights and inputs are random: this shows the calls and their order, not a trained network.
"""

from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass
from pathlib import Path

import torch

if str(Path(__file__).resolve().parent.parent) not in sys.path:
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from jasnamacos_b200 import synthetic  # noqa: E402
from jasnamacos_b200.deform_conv import CudaDeformConv, DeformConvShape  # noqa: E402
from jasnamacos_b200.token_ops import CudaTokenOps  # noqa: E402

PATCH, SIDE, CHANNELS = 4, 64, 64
TOKENS = (SIDE // PATCH) ** 2  # of a frame
WIDTH = CHANNELS * PATCH * PATCH
HEADS, KV_HEADS, HEAD_DIM = 16, 4, 64
PAIRS = (8, 12, 12)  # of a head, for (time, row, column)


@dataclass
class Weights:
    norm1: torch.Tensor
    norm2: torch.Tensor
    norm3: torch.Tensor
    qkv: torch.Tensor
    out: torch.Tensor
    up: torch.Tensor
    down: torch.Tensor
    modulation: torch.Tensor  # [streams][6][WIDTH]: shift, scale, gate of attention, then of the MLP

    @classmethod
    def random(cls, streams: int, seed: int = 0) -> "Weights":
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, scale):
            return (torch.randn(shape, generator=g, device="cuda") * scale).half()

        return cls(1 + normal(WIDTH, scale=0.1), 1 + normal(WIDTH, scale=0.1), 1 + normal(WIDTH, scale=0.1),
                   normal(WIDTH, (HEADS + 2 * KV_HEADS) * HEAD_DIM, scale=WIDTH ** -0.5),
                   normal(HEADS * HEAD_DIM, WIDTH, scale=WIDTH ** -0.5), normal(WIDTH, 2 * WIDTH, scale=WIDTH ** -0.5),
                   normal(2 * WIDTH, WIDTH, scale=WIDTH ** -0.5), normal(streams, 6, WIDTH, scale=0.3))


class FrameStream:
    """The block's state for `streams` streams that take frames together."""

    def __init__(self, weights: Weights, streams: int, window: int = 8, sinks: int = 1):
        self.ops = CudaTokenOps()
        self.w, self.streams, self.window, self.sinks = weights, streams, window, sinks
        self.frame = 0
        pages = sinks + window  # of a stream
        self.k_cache = torch.zeros(streams * pages, TOKENS, KV_HEADS, HEAD_DIM, dtype=torch.float16, device="cuda")
        self.v_cache = torch.zeros_like(self.k_cache)
        # Frame f's page: the first frames keep theirs, the others take turns.  Frames from sinks + window on see the
        # first frames and a whole window behind them, so their places in the stream repeat with their pages.
        f = torch.arange(sinks + 2 * window, device="cuda")
        page = torch.where(f < sinks, f, sinks + (f - sinks) % window)
        self.table = (page + pages * torch.arange(streams, device="cuda")[:, None]).int().contiguous()
        self.starts = (TOKENS * torch.arange(streams + 1, device="cuda")).int()
        self.lengths = torch.zeros(streams, dtype=torch.int32, device="cuda")
        row, column = torch.meshgrid(*[torch.arange(SIDE // PATCH, device="cuda")] * 2, indexing="ij")
        place = torch.stack([torch.zeros_like(row), row, column], -1).view(1, TOKENS, 3)
        self.positions = place.expand(streams, -1, -1).reshape(-1, 3).int().contiguous()
        series = [10000.0 ** (-i / n) for n in PAIRS for i in range(n)]
        self.frequencies = torch.tensor(series, dtype=torch.float64, device="cuda")

    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """One frame of every stream: tokens [streams * TOKENS, WIDTH] FP16 in and out."""
        ops, w = self.ops, self.w
        shift1, scale1, gate1, shift2, scale2, gate2 = w.modulation.unbind(1)
        place = self.frame
        if place >= self.sinks + self.window:
            place = self.sinks + self.window + (place - self.sinks) % self.window
        self.positions[:, 0] = self.frame
        self.frame += 1
        self.lengths.fill_((place + 1) * TOKENS)

        x = ops.norm(tokens, kind="layer", weight=w.norm1, scale=scale1, shift=shift1, group=TOKENS)
        qkv = (x @ w.qkv).view(-1, HEADS + 2 * KV_HEADS, HEAD_DIM)
        q, k, v = qkv.split((HEADS, KV_HEADS, KV_HEADS), 1)
        q = ops.append(k, v, self.k_cache, self.v_cache, self.table, self.starts, self.lengths, q=q, positions=self.positions,
                       frequencies=self.frequencies, pairs=PAIRS)
        attended = ops.attention(q, self.k_cache, self.v_cache, self.table, self.starts, self.lengths, max_q=TOKENS,
                                 max_kv=(place + 1) * TOKENS, window=self.window, sinks=self.sinks, frame=TOKENS)
        tokens, x = ops.residual_norm(attended.view(-1, HEADS * HEAD_DIM) @ w.out, tokens, gate=gate1, kind="layer",
                                      weight=w.norm2, scale=scale2, shift=shift2, group=TOKENS)
        x = torch.nn.functional.silu(x @ w.up) @ w.down
        # The norm that follows belongs to the next block; here it is left unused but for its place in the pass.
        tokens, _ = ops.residual_norm(x, tokens, gate=gate2, kind="layer", weight=w.norm3, group=TOKENS)
        return tokens


def patches(features: torch.Tensor) -> torch.Tensor:
    """[streams][CHANNELS][SIDE][SIDE] -> [streams * TOKENS][WIDTH]."""
    n, side = features.shape[0], SIDE // PATCH
    cut = features.view(n, CHANNELS, side, PATCH, side, PATCH)
    return cut.permute(0, 2, 4, 1, 3, 5).reshape(n * TOKENS, WIDTH)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--streams", type=int, default=8)
    ap.add_argument("--frames", type=int, default=30)
    args = ap.parse_args()
    dcn = CudaDeformConv()
    shape = DeformConvShape.jasna_propagation(args.streams)
    weight, bias = synthetic.weights(shape, 1)
    packed = dcn.prepack(shape, torch.from_numpy(weight).cuda().half())
    bias = torch.from_numpy(bias).cuda().half()
    block = FrameStream(Weights.random(args.streams), args.streams)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for f in range(args.frames):
        x, offset, mask, _, _ = synthetic.device_batch(shape, 16.0, seed=f, device="cuda")
        if f == args.frames // 2:
            begin.record()
        aligned = dcn.forward_f16(shape, x, offset, mask, packed, bias)
        tokens = block.step(patches(aligned.view(args.streams, CHANNELS, SIDE, SIDE)))
        if f == args.frames // 2:
            end.record()
    torch.cuda.synchronize()
    dcn.device_error()
    print(f"{args.streams} streams, {args.frames} frames: output {tuple(tokens.shape)}, finite: {bool(tokens.isfinite().all())}; "
          f"frame {args.frames // 2}: {begin.elapsed_time(end):.3f} ms (alignment and block)")


if __name__ == "__main__":
    main()
