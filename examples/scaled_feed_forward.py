"""A feed-forward block on block-scaled 8-bit weights: norm with the residual's
addition -> product -> gate -> encode -> product, for one token or a batch.

    python examples/scaled_feed_forward.py [--tokens 1] [--width 4096] [--inner 8192]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from accessor_universal_test_b200 import Workspace, scaled  # noqa: E402


class FeedForward:
    """Weights are encoded once; every call reads one byte of them a value."""

    def __init__(self, ws: Workspace, gain: torch.Tensor, up: torch.Tensor, down: torch.Tensor):
        """gain [width], up [2 inner, width], down [width, inner]."""
        self.ws, self.gain = ws, gain
        self.up = scaled.encode(ws, up, block_rows=128)
        self.down = scaled.encode(ws, down, block_rows=128)

    def __call__(self, x: torch.Tensor, stream: torch.Tensor) -> torch.Tensor:
        """x [tokens, width] joins `stream` (in place); returns the block's part."""
        a, _ = scaled.rms_norm(self.ws, x, self.gain, residual=stream)
        gate, value = scaled.matmul(self.ws, a, self.up, dtype=x.dtype).chunk(2, dim=1)
        h = scaled.encode(self.ws, torch.nn.functional.silu(gate) * value)
        return scaled.matmul(self.ws, h, self.down, dtype=x.dtype)


def reference(gain, up, down, x, stream):
    """The block in FP32 without 8-bit codes."""
    h = x.float() + stream.float()
    a = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-5) * gain.float()
    gate, value = (a @ up.float().t()).chunk(2, dim=1)
    return (torch.nn.functional.silu(gate) * value) @ down.float().t(), h


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=1)
    ap.add_argument("--width", type=int, default=4096)
    ap.add_argument("--inner", type=int, default=8192)
    args = ap.parse_args()
    g = torch.Generator(device="cuda").manual_seed(1)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16()

    gain = 1 + normal(args.width, scale=0.1)
    up = normal(2 * args.inner, args.width, scale=args.width ** -0.5)
    down = normal(args.width, args.inner, scale=args.inner ** -0.5)
    x, stream = normal(args.tokens, args.width), normal(args.tokens, args.width)
    want, _ = reference(gain, up, down, x, stream)
    ws = Workspace(0)
    block = FeedForward(ws, gain, up, down)
    got = block(x, stream.clone())
    error = (got.float() - want).norm() / want.norm()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    repeats = 20
    for _ in range(3):
        block(x, stream)
    begin.record()
    for _ in range(repeats):
        block(x, stream)
    end.record()
    torch.cuda.synchronize()
    print(f"{args.tokens} tokens, {args.width} -> 2 x {args.inner} -> {args.width}: "
          f"{begin.elapsed_time(end) / repeats * 1e3:.1f} us, relative error against FP32 {error:.4f}")
    ws.close()


if __name__ == "__main__":
    main()
