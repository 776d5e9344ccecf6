"""A rewind that is refused leaves the cache as it was."""
import pytest
import torch

from nanokv_b200.block_cache import BlockCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[64.0, 64], [64, 64.0], [0, "1"], [128, None]])
def test_lengths_that_are_no_integers(lengths):
    cache = BlockCache(2, 1, 64, 512)
    k = torch.randn(2, 130, 1, 64, device="cuda").to(torch.bfloat16)
    cache.append(k, k)
    cache.weights.fill_(1.0)
    with pytest.raises(TypeError):
        cache.rewind(lengths)
    assert cache.lengths == [130, 130] and bool((cache.weights == 1.0).all())
    cache.append(k[:, :3], k[:, :3])
    assert cache.lengths == [133, 133]
    again = cache.read(128, 133)[0]
    assert torch.equal(again[:, :2], k[:, 128:]) and torch.equal(again[:, 2:], k[:, :3])
    cache.rewind([130, 129])
    assert cache.lengths == [130, 129]
