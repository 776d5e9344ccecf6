"""Host integers that a call cannot pass on as they are."""
import pytest
import torch

from nanokv_b200 import ops


@pytest.mark.parametrize("value", [2 ** 31, 2 ** 32 + 3, -2 ** 31 - 1, 2 ** 70])
def test_integers_past_32_bits_are_refused(value):
    with pytest.raises(ValueError, match="counts"):
        ops._host_ints([1, value], 2, "counts")
    with pytest.raises(ValueError, match="keep"):
        ops._int32(value, "keep")


def test_integers_of_32_bits_pass():
    assert list(ops._host_ints([2 ** 31 - 1, -2 ** 31, 0], 3, "counts")) == [2 ** 31 - 1, -2 ** 31, 0]
    assert list(ops._host_ints([], 0, "counts")) == [] and ops._host_ints(None, 4, "counts") is None
    assert ops._int32(2 ** 31 - 1, "keep") == 2 ** 31 - 1


@pytest.mark.gpu
def test_calls_that_are_refused_leave_the_cache_as_it_was():
    from nanokv_b200.block_cache import BlockCache
    cache = BlockCache(2, 1, 64, 512)
    k = torch.randn(2, 130, 1, 64, device="cuda").to(torch.bfloat16)
    cache.append(k, k)
    cache.weights.fill_(1.0)
    table = cache.table.clone()
    for call in (lambda: cache.append(k, k, counts=[2 ** 32 + 3, 1]), lambda: cache.attend(k, counts=[2 ** 32, 1]),
                 lambda: cache.read(2 ** 32, 2 ** 32 + 1), lambda: cache.evict(2 ** 32, sinks=0, recent=0),
                 lambda: cache.evict(2 ** 32 + 1, sinks=1, recent=2 ** 32)):
        with pytest.raises(ValueError):
            call()
    assert cache.lengths == [130, 130] and torch.equal(cache.table, table) and bool((cache.weights == 1.0).all())
    cache.append(k[:, :3], k[:, :3])
    assert cache.lengths == [133, 133]
    again = cache.read(128, 133)[0]
    assert torch.equal(again[:, :2], k[:, 128:]) and torch.equal(again[:, 2:], k[:, :3])
