"""Stored codes against the quotient they are defined by, for every 16-bit number under every largest magnitude."""
import pytest
import torch

from nanokv_b200.block_cache import BLOCK, BlockCache

pytestmark = pytest.mark.gpu
SIDE = BLOCK * BLOCK       # elements of a block of 64-wide heads


@pytest.mark.parametrize("dtype,finite", [(torch.bfloat16, 0x7F80), (torch.float16, 0x7C00)])
def test_codes_are_the_rounded_quotients(dtype, finite):
    """Blocks of one kv head each: the head's number is the bits of its largest magnitude, the block's other elements are
    consecutive magnitudes up to it, of either sign.  scale = largest / 127 and x / scale are fp32 quotients, rounded to
    nearest; the code is the nearest integer, ties to even, in -127 .. 127."""
    for first in range(0, finite, SIDE - 1):
        # magnitudes first .. first + SIDE - 2, under every largest one that is not below `first`
        most = torch.arange(max(1, first), finite, device="cuda")
        bits = torch.minimum(first + torch.arange(SIDE - 1, device="cuda"), most[:, None])
        x = torch.cat([most[:, None], bits], 1).to(torch.int16).view(dtype)
        x = torch.where(torch.arange(SIDE, device="cuda") % 3 == 1, -x, x)
        heads = len(most)
        rows = x.view(heads, BLOCK, BLOCK).transpose(0, 1)[None]
        cache = BlockCache(1, heads, BLOCK, BLOCK, dtype=dtype)
        cache.append(rows, -rows)
        scale = x[:, :1].float().abs() / torch.full((1, 1), 127.0, device="cuda")
        assert torch.equal(cache.scales[0, :, 0], scale.expand(heads, 2))
        want = torch.round(x.float() / scale).clamp_(-127, 127) + 128
        assert torch.equal(cache.k_codes.view(heads, SIDE).float(), want)
        assert torch.equal(cache.v_codes[0, :, 0].transpose(1, 2).reshape(heads, SIDE).float(), 256 - want)
