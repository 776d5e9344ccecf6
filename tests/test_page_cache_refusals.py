"""Calls of the paged cache that would write one place twice, or take what is no number: refused on the host, no GPU needed."""
import pytest
import torch

from nanokv_b200 import _lib
from test_page_cache_host import HostTable, on_host, rows, status_of, struct  # noqa: F401


def test_pools_that_are_written_twice():
    """One pool as keys and values of a cache that is written, or of two caches of a call."""
    one = struct(address=1024, v=1024)
    status, text = status_of("nkv_page_append", one, rows(2), rows(2), None, None, 1, None, None, 256, None)
    assert status == _lib.NKV_ERR_INVALID and "one pool" in text
    crossed = (_lib.PageCache * 2)(struct(address=1024, v=2048), struct(address=2048, v=4096))
    for caches, count in (((_lib.PageCache * 1)(one), 1), (crossed, 2)):
        status, text = status_of("nkv_page_keep", caches, count, 256, 1, None, 256, None)
        assert status == _lib.NKV_ERR_INVALID and "are one" in text


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
def test_scales_that_are_no_number_in_base_two(scale):
    """The kernels take scale * log2(e)."""
    status, text = status_of("nkv_page_attend", struct(), rows(2), 1, None, None, 0, 1, scale, 256, 256, 256, None, 0, None)
    assert status == _lib.NKV_ERR_INVALID and "finite" in text


def test_a_sequence_named_by_another_integer_type(on_host):  # noqa: F811
    """What indexes a list and what indexes a tensor are not the same: True is sequence 1 of both, 1.0 of neither."""
    table = HostTable(3, 100, 12, 16)
    table.reserve([40, 50, 60])
    table.release(True)
    assert (table.table[1] == -1).all() and (table.table[0, :3] >= 0).all() and (table.table[2, :4] >= 0).all()
    assert table.free == 12 - 3 - 4
    table.release(torch.tensor(2))
    assert (table.table[2] == -1).all() and table.free == 12 - 3
    for sequence in (0.0, "0", None):
        with pytest.raises(TypeError):
            table.release(sequence)
    assert table.free == 12 - 3 and (table.table[0, :3] >= 0).all()
