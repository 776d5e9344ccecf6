"""Rotation, append, attention and eviction together, as a decoder uses them, against the formulas in 64 bits."""
import sys
from pathlib import Path

import pytest
import torch

import block_reference as ref
from nanokv_b200 import ops

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

pytestmark = pytest.mark.gpu


def test_a_stream_with_evictions():
    from stream_block_cache import Stream
    batch, heads, kv_heads, dim, keep = 2, 4, 2, 64, 4
    stream = Stream(batch, heads, kv_heads, dim, (keep + 4) * 64, keep=keep, recent=1, positions=1024)
    gen = torch.Generator().manual_seed(3)
    table = stream.rotary.table.cpu()
    held_k = [[torch.zeros(0, dim, dtype=torch.float64) for _ in range(kv_heads)] for _ in range(batch)]
    held_v = [[torch.zeros(0, dim, dtype=torch.float64) for _ in range(kv_heads)] for _ in range(batch)]
    seen = 0
    for tokens in [150, 1, 1, 60, 1, 120, 1, 63, 1]:
        q, k, v = (torch.randn(batch, tokens, h, dim, generator=gen).to(torch.bfloat16) for h in (heads, kv_heads, kv_heads))
        out, lse = stream.step(q.cuda(), k.cuda(), v.cuda())
        ops.check_status(out.device)
        positions = torch.arange(seen, seen + tokens, dtype=torch.int32).expand(batch, tokens)
        seen += tokens
        # fp32 rotation and 64-bit rotation round to the same bf16 number but for a few: what the cache holds is checked with
        # the rotation's own test, here its rows are taken as they are
        turned = stream.rotary.apply(k.cuda(), positions=positions.contiguous().cuda()).cpu().double()
        q_turned = ref.rotated(q, table, positions, "half").to(torch.bfloat16)
        for b in range(batch):
            for h in range(kv_heads):
                held_k[b][h] = torch.cat([held_k[b][h], turned[b, :, h]])
                held_v[b][h] = torch.cat([held_v[b][h], v[b, :, h].double()])
                full = held_k[b][h].shape[0] // 64
                # full blocks as the cache holds them (quantising twice changes nothing: the largest element of a block is a code)
                for i in range(full):
                    for rows in (held_k, held_v):
                        rows[b][h][64 * i:64 * i + 64] = ref.quantised(rows[b][h][64 * i:64 * i + 64, None])[:, 0]
        keys, values = (torch.stack([torch.stack(row, 1) for row in rows]) for rows in (held_k, held_v))
        lengths = [keys.shape[1]] * batch
        want, want_lse, spread, size, _ = ref.attention(q_turned, keys, values, lengths, [tokens] * batch, True, dim ** -0.5)
        # queries may differ by one rounding of the rotation: 2^-8 of the scores' magnitudes, besides the kernel's own bounds
        score = 2.0 ** -8 * size.clamp_min(1.0)
        assert ((lse.double().cpu() - want_lse).abs() <= score).all()
        assert ((out.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -7 + 4 * score[..., None]) * spread).all()
        # follow the cache's own choice of blocks
        if stream.cache.lengths != lengths:
            assert stream.cache.lengths == [keep * 64 + lengths[0] % 64] * batch
            got_k, _ = stream.cache.read(0, stream.cache.lengths[0])
            got_k = got_k.double().cpu()
            for b in range(batch):
                for h in range(kv_heads):
                    blocks = held_k[b][h].shape[0] // 64
                    kept = [i for i in range(blocks) if any(
                        float((got_k[b, 64 * j:64 * j + 64, h] - held_k[b][h][64 * i:64 * i + 64]).abs().max()) < 0.05 for j in range(keep))]
                    assert len(kept) == keep and kept[0] == 0 and kept[-1] == blocks - 1
                    for rows in (held_k, held_v):
                        parts = [rows[b][h][64 * i:64 * i + 64] for i in kept] + [rows[b][h][64 * blocks:]]
                        rows[b][h] = torch.cat(parts)
    assert stream.cache.lengths[0] < seen
