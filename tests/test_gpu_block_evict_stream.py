"""Eviction on a stream that the cache's arrays do not come from."""
import pytest
import torch

from nanokv_b200.block_cache import BlockCache

pytestmark = pytest.mark.gpu


def test_memory_of_a_table_is_not_handed_out_while_its_eviction_waits():
    """The cache lets go of its table and weights; the allocator must not give them to the stream they came from while the
    eviction that reads them is still to run on another."""
    cache = BlockCache(2, 4, 64, 64 * 300)
    cache.append(*(torch.randn(2, 64 * 20, 4, 64, device="cuda").to(torch.bfloat16) for _ in range(2)))
    cache.weights.copy_(torch.rand_like(cache.weights))
    weights, table = cache.weights.tolist(), cache.table.tolist()
    held = cache.table.data_ptr(), cache.weights.data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)         # a tenth of a second
        cache.evict(8, sinks=1, recent=1)
    late = side.record_event()
    taken = [torch.empty(2, 4, 300, dtype=torch.int32, device="cuda") for _ in range(8)]
    assert not late.query()                    # the eviction is still to run
    assert not {t.data_ptr() for t in taken} & set(held)
    torch.cuda.synchronize()
    assert cache.lengths == [64 * 8] * 2
    for b in range(2):
        for h in range(4):
            middle = sorted(range(1, 19), key=lambda i: -weights[b][h][i])[:6]
            kept = sorted([0, 19, *middle])
            assert cache.table[b, h, :8].tolist() == [table[b][h][i] for i in kept]
            assert cache.weights[b, h, :8].tolist() == [weights[b][h][i] for i in kept]
