"""Chunks appended behind an open block, which complete it and leave another, against the same tokens one at a time."""
import pytest
import torch

from nanokv_b200.block_cache import BlockCache
from nanokv_b200.rotary import Rotary

pytestmark = pytest.mark.gpu


def rows(*shape, seed, dtype):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def cache_of(batch, heads, dim, dtype):
    cache = BlockCache(batch, heads, dim, 512, dtype=dtype)
    for name in ("k_codes", "v_codes", "scales", "k_tail", "v_tail"):
        getattr(cache, name).zero_()
    return cache


def same(a, b):
    assert a.lengths == b.lengths
    for name in ("k_codes", "v_codes", "scales"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    for i, n in enumerate(a.lengths):
        open_rows = n % 64
        assert torch.equal(a.k_tail[i, :, :open_rows], b.k_tail[i, :, :open_rows]), i
        assert torch.equal(a.v_tail[i, :, :, :open_rows], b.v_tail[i, :, :, :open_rows]), i


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rotary", [None, "half", "interleaved"])
@pytest.mark.parametrize("batch,heads,start", [(3, 2, 1), (32, 40, 30), (32, 40, 63)])
def test_a_chunk_across_blocks_is_its_tokens_one_by_one(batch, heads, start, rotary, dim, dtype):
    """All sequences and heads complete a block from old and new rows and open another, in one call and then in more."""
    chunks = [start, 64, 130, 50]
    total = sum(chunks)
    k, v = (rows(batch, total, heads, dim, seed=s, dtype=dtype) for s in (1, 2))
    keywords = {}
    if rotary:
        keywords["rotary"] = Rotary(dim, total, layout=rotary)
    positions = torch.arange(total, dtype=torch.int32, device="cuda").expand(batch, total)

    def put(cache, at, n):
        more = dict(positions=positions[:, at:at + n].contiguous()) if rotary else {}
        cache.append(k[:, at:at + n], v[:, at:at + n], **keywords, **more)

    single, chunked = cache_of(batch, heads, dim, dtype), cache_of(batch, heads, dim, dtype)
    at = 0
    for n in chunks:
        put(chunked, at, n)
        for t in range(at, at + n):
            put(single, t, 1)
        at += n
        same(chunked, single)


def test_sequences_that_do_and_do_not_cross_in_one_call():
    """Counts of their own: some sequences cross a block's end, some stop at it, some stay inside, some take nothing, over more
    sequences than a launch has."""
    batch, heads, dim = 150, 3, 128
    starts, counts = [(37 * i) % 130 for i in range(batch)], [(53 * i) % 140 for i in range(batch)]
    starts[:4], counts[:4] = [30, 32, 0, 63], [98, 32, 64, 1]
    k, v = (rows(batch, 280, heads, dim, seed=s, dtype=torch.bfloat16) for s in (3, 4))
    single, chunked = cache_of(batch, heads, dim, torch.bfloat16), cache_of(batch, heads, dim, torch.bfloat16)
    chunked.append(k[:, :140], v[:, :140], counts=starts)
    chunked.append(k[:, 140:], v[:, 140:], counts=counts)
    for wanted, at in ((starts, 0), (counts, 140)):
        for t in range(140):
            single.append(k[:, at + t:at + t + 1], v[:, at + t:at + t + 1], counts=[int(t < n) for n in wanted])
    same(chunked, single)
