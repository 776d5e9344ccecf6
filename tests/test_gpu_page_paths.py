"""Accepted paths with nodes that cannot be followed, and what captured calls report."""
import pytest
import torch

import page_reference as ref
from nanokv_b200 import ops, page_cache
from nanokv_b200.page_cache import PageCache, PageTable

pytestmark = pytest.mark.gpu


def moved(pool, table, lengths, paths, counts, tokens):
    """The pool after the nodes of the paths that can be followed: ascending, none ahead of the place it moves to."""
    out = pool.clone()
    for b, (n, c) in enumerate(zip(lengths, counts)):
        rows, before = ref.rows_of(pool, table, b, n + tokens), -1
        for j, node in enumerate(paths[b][:c]):
            if before < node and j <= node < tokens:
                before = node
                ref.put(out, table, b, n + j, rows[n + node][None])
    return out


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("path", [[-1, 0, 1, 2, 3, 4, 5, 6, 7, 8], [0, 0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16], [3, -1, 5, 2, 7, 9, 9, 10, 11, 30],
                                  [2, 2, 2, 2, 2, 2, 2, 2, 2, 2, 11], [31, 1, 2, 3, 4, 5, 6, 7, 8, 9], [-5, -4, -3, -2, -1, 0, 1, 2, 3, 4, 20, 21]])
def test_a_node_that_cannot_be_followed_moves_nothing(path, page):
    """In a path of more rows than a thread has in flight: rows that others move to are not read afterwards."""
    lengths, tokens, heads, D = [5, 40, 0], 32, 2, 64
    table, pages = ref.scattered(3, 80, page, 3)
    k, v = (ref.randn(pages, heads, page, D, seed=s, dtype=torch.bfloat16) for s in (1, 2))
    good = list(range(2, 2 + len(path)))
    paths, counts = [path, good, path], [len(path), len(path), len(path) - 1]
    pt = PageTable.over(table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), pages=pages, page=page)
    caches = [PageCache.over(pt, k.cuda(), v.cuda()) for _ in range(2)]
    page_cache.keep(caches, torch.tensor(paths, dtype=torch.int32).cuda(), torch.tensor(counts, dtype=torch.int32).cuda())
    with pytest.raises(RuntimeError, match="path out of range"):
        ops.check_status("cuda:0")
    for cache in caches:
        for got, pool in ((cache.k_pages, k), (cache.v_pages, v)):
            assert torch.equal(got.cpu(), moved(pool, table, lengths, paths, counts, tokens))


def test_a_captured_tree_mask_does_not_clear_what_others_report(monkeypatch):
    """Captured before anything on the device has reported: the graph must not hold the device's status word, which each replay would clear."""
    monkeypatch.setattr(ops, "_STATUS_WORDS", {})
    parents = torch.tensor([-1, 0, 0, 2], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mask, depth = ops.tree_mask(parents)
    ops.tree_mask(torch.tensor([3], dtype=torch.int32, device="cuda"))       # reports its parent
    graph.replay()
    assert mask.flatten().tolist() == [1, 3, 5, 13] and depth.tolist() == [0, 1, 1, 2]
    with pytest.raises(RuntimeError, match="parent"):
        ops.check_status("cuda:0")


def test_a_captured_tree_mask_reports_where_there_is_a_word():
    ops.status_word(torch.device("cuda:0"))
    parents = torch.tensor([-1, 0], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mask, _ = ops.tree_mask(parents)
    graph.replay()
    ops.check_status("cuda:0")
    parents[1] = 1
    graph.replay()
    assert mask.flatten().tolist() == [1, 2]
    with pytest.raises(RuntimeError, match="parent"):
        ops.check_status("cuda:0")


def test_a_captured_keep_reports_into_its_tables_word(monkeypatch):
    table = PageTable(1, 64, pages=4, page=16)
    table.reserve([40])
    cache = PageCache(table, 1, 64)
    x = ref.randn(1, 8, 1, 64, seed=1, dtype=torch.bfloat16).cuda()
    cache.append(x, x)
    path = torch.tensor([[1, 3]], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    word = table.status
    monkeypatch.setattr(ops, "_STATUS_WORDS", {})
    with torch.cuda.graph(graph):
        cache.keep(path)
    path[0, 1] = 0
    graph.replay()
    torch.cuda.synchronize()
    assert int(word) == 920 and not ops._STATUS_WORDS
    word.zero_()


def test_the_first_table_is_not_made_inside_a_capture(monkeypatch):
    table, lengths = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    kept = torch.ones(1, device="cuda")
    monkeypatch.setattr(ops, "_STATUS_WORDS", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept.add_(1)
        with pytest.raises(RuntimeError, match="outside a graph capture"):
            PageTable.over(table, lengths, pages=4, page=16)
    assert not ops._STATUS_WORDS
    graph.replay()
    assert float(kept) == 2
    PageTable.over(table, lengths, pages=4, page=16)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        kept.add_(1)
        PageTable.over(table, lengths, pages=4, page=16)
