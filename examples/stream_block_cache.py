"""Sequences streamed through an 8-bit block cache: a prompt in chunks, then token by token, with room made as it fills.

    python examples/stream_block_cache.py [--batch B] [--prompt N] [--tokens N] [--keep BLOCKS]

One layer's cache as a decoder would use it: queries and keys are rotated by their positions (a table scaled for long
contexts), keys and values are appended, the queries attend with the weight of every block added up, and whenever a
sequence holds more than ``--keep`` full blocks, those that attention used least are freed for its kv head.  Queries, keys
and values are random: there is no model here.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from nanokv_b200.block_cache import BLOCK, BlockCache  # noqa: E402
from nanokv_b200.rotary import Rotary  # noqa: E402


class Stream:
    """The cache and rotation of one layer; ``step`` takes the next tokens of every sequence."""

    def __init__(self, batch: int, heads: int, kv_heads: int, head_dim: int, capacity: int, *, keep: int, recent: int = 4,
                 positions: int = 32768, dtype: torch.dtype = torch.bfloat16):
        self.cache = BlockCache(batch, kv_heads, head_dim, capacity, dtype=dtype)
        self.rotary = Rotary(head_dim, positions, scaling=dict(kind="blend", factor=4.0, trained=8192), device=self.cache.device)
        self.heads, self.keep, self.recent, self.seen = heads, keep, recent, 0

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
        """q [batch, tokens, heads, head_dim], k and v [batch, tokens, kv_heads, head_dim] -> (O, lse)."""
        batch, tokens = q.shape[:2]
        positions = torch.arange(self.seen, self.seen + tokens, dtype=torch.int32, device=q.device).expand(batch, tokens).contiguous()
        self.seen += tokens
        # the keys are rotated as they are stored; positions go on counting when blocks leave
        self.cache.append(k, v, rotary=self.rotary, positions=positions)
        out, lse = self.cache.attend(self.rotary.apply(q, positions=positions), weights=self.cache.weights)
        if max(self.cache.lengths) // BLOCK > self.keep:
            self.cache.evict(self.keep, sinks=1, recent=self.recent)
        return out, lse


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--batch", type=int, default=4)
    parser.add_argument("--prompt", type=int, default=4680)
    parser.add_argument("--tokens", type=int, default=400)
    parser.add_argument("--keep", type=int, default=64)
    args = parser.parse_args()
    heads, kv_heads, dim, chunk = 40, 8, 128, 1560
    stream = Stream(args.batch, heads, kv_heads, dim, (args.keep + 2) * BLOCK + chunk, keep=args.keep)
    gen = torch.Generator(device="cuda").manual_seed(0)

    def rows(tokens, h):
        return torch.randn(args.batch, tokens, h, dim, generator=gen, device="cuda").to(torch.bfloat16)

    for start in range(0, args.prompt, chunk):
        n = min(chunk, args.prompt - start)
        stream.step(rows(n, heads), rows(n, kv_heads), rows(n, kv_heads))
    inputs = rows(1, heads), rows(1, kv_heads), rows(1, kv_heads)
    torch.cuda.synchronize()
    begin = time.perf_counter()
    for _ in range(args.tokens):
        out, lse = stream.step(*inputs)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - begin
    print(f"{args.batch} sequences: {args.prompt} prompt tokens, then {args.tokens} one by one at {seconds / args.tokens * 1e6:.0f} us; "
          f"{stream.cache.lengths[0]} tokens held of {stream.seen}, largest |O| {float(out.abs().max()):.3f}")


if __name__ == "__main__":
    main()
