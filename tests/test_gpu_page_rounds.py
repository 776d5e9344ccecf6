"""Attention over the paged cache where thread blocks take several runs of the list, and calls at the edges of what is allowed."""
import math

import pytest
import torch

import page_reference as ref
from nanokv_b200 import ops
from nanokv_b200.page_cache import PageCache, PageTable

pytestmark = pytest.mark.gpu


def over(k, v, table, lengths, page):
    pt = PageTable.over(table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), pages=k.shape[0], page=page)
    return PageCache.over(pt, k, v)


def on_gpu(q, k, v, seen, scale):
    """One head's queries [n, D] over the first seen[i] of rows k, v [N, D], in 64 bits -> out, lse, spread, size."""
    s = q.double() @ k.double().T * scale
    hidden = torch.arange(k.shape[0], device=q.device) >= seen[:, None]
    total = torch.logsumexp(s.masked_fill(hidden, -math.inf), -1)
    p = torch.exp(s - total[:, None]).masked_fill(hidden, 0.0)
    size = (q.double().abs() @ k.double().abs().T * scale).masked_fill(hidden, 0.0).amax(-1)
    return p @ v.double(), total, p @ v.double().abs(), size


@pytest.mark.parametrize("dtype,D,heads,tokens,length", [(torch.bfloat16, 128, 8, 2300, 33000), (torch.float16, 64, 8, 2000, 42000)])
def test_several_rounds_of_runs(dtype, D, heads, tokens, length):
    """Keys and values of more than 64 MB, so many units that a block's run is cut: rows at the borders of units and pages."""
    page, total = 128, length + tokens
    gen = torch.Generator(device="cuda").manual_seed(1)
    pages = -(-total // page) + 2
    k, v = (torch.randn(pages, heads, page, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
    table = torch.randperm(pages, generator=gen, device="cuda")[:pages - 2].to(torch.int32)[None].contiguous()
    cache = over(k, v, table, [length], page)
    q = torch.randn(1, tokens, heads, D, generator=gen, device="cuda").to(dtype)
    assert 4 * D * heads * total > 64 << 20
    out, lse = cache.attend(q)
    ops.check_status("cuda:0")
    again, lse_again = cache.attend(q)
    assert torch.equal(out, again) and torch.equal(lse, lse_again)
    rows = torch.tensor(sorted({0, 1, 127, 128, 255, 256, 257, tokens // 2, tokens - 257, tokens - 129, tokens - 1}), device="cuda")
    unit = ref.UNIT[dtype]
    for h in range(heads):
        kh, vh = (pool[table[0].long(), h].reshape(-1, D)[:total] for pool in (k, v))
        want, total_lse, spread, size = on_gpu(q[0, rows, h], kh, vh, length + rows + 1, D ** -0.5)
        score = 2.0 ** -18 * size.clamp_min(1.0)
        # as in test_gpu_page_cache: rounding of the result and of the weights, fp32 scores, fp32 sums (of independent roundings: 2^-12 of
        # them over 42,000 tokens), fp16 weights of half a step of 2^-25 where the largest has 2^7
        bound = unit * want.abs() + (2 * unit + 4 * score[:, None] + 2.0 ** -12) * spread + 1e-7
        if dtype == torch.float16:
            bound = bound + 2.0 ** -32 * total * float(vh.abs().max())
        assert ((out[0, rows, h].double() - want).abs() <= bound).all()
        assert ((lse[0, rows, h].double() - total_lse).abs() <= score + 2.0 ** -12).all()


@pytest.mark.parametrize("group,tokens", [(320, 1), (129, 2), (64, 4)])
def test_many_query_heads_to_a_kv_head(group, tokens):
    lengths = [5, 400]
    table, pages = ref.scattered(2, 410, 32, 3)
    k, v = (ref.randn(pages, 1, 32, 64, seed=s, dtype=torch.bfloat16) for s in (1, 2))
    cache = over(k.cuda(), v.cuda(), table.cuda(), lengths, 32)
    q = ref.randn(2, tokens, group, 64, seed=4, dtype=torch.bfloat16)
    out, lse = cache.attend(q.cuda())
    ops.check_status("cuda:0")
    mask = torch.ones(2, tokens, tokens, dtype=torch.bool).tril()
    want, want_lse, spread, size = ref.attention(q, k, v, table, lengths, [tokens] * 2, mask, 0.125)
    unit, score = ref.UNIT[torch.bfloat16], 2.0 ** -18 * size.clamp_min(1.0)
    assert ((lse.double().cpu() - want_lse).abs() <= score + 2.0 ** -13).all()
    assert ((out.double().cpu() - want).abs() <= unit * want.abs() + (2 * unit + 4 * score[..., None] + 2.0 ** -13) * spread + 1e-7).all()


def test_rows_shared_by_heads_and_sequences():
    """Queries, keys and values that are one row expanded: strides of zero."""
    one = ref.randn(1, 1, 1, 64, seed=1, dtype=torch.float16).cuda()
    k, v = (torch.zeros(6, 2, 16, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.arange(6, dtype=torch.int32, device="cuda").reshape(2, 3)
    cache = over(k, v, table, [0, 0], 16)
    cache.append(one.expand(2, 40, 2, 64), one.expand(2, 40, 2, 64))
    out, lse = cache.attend(one.expand(2, 40, 8, 64))
    ops.check_status("cuda:0")
    assert ((out - one).abs() <= 2 * ref.UNIT[torch.float16] * one.abs() + 1e-7).all()
    s = float((one.double() ** 2).sum() / 8)
    want = s + torch.log(torch.arange(1, 41, dtype=torch.float64, device="cuda"))
    assert ((lse.double() - want[None, :, None]).abs() <= 2.0 ** -16 * max(1.0, s)).all()


def test_two_graphs_of_one_cache_replayed_in_turn():
    """A step of one token and one of a draft, captured apart; the lengths they find are those of the replay."""
    table = PageTable(2, 400, pages=40, page=32)
    table.reserve([400, 300])
    cache = PageCache(table, 2, 64, dtype=torch.bfloat16)
    k, v = (ref.randn(2, 200, 2, 64, seed=s, dtype=torch.bfloat16).cuda() for s in (1, 2))
    cache.append(k, v)
    table.advance(200)
    small, large = (ref.randn(2, t, 8, 64, seed=t, dtype=torch.bfloat16).cuda() for t in (1, 70))
    new_small, new_large = (ref.randn(2, t, 2, 64, seed=t + 1, dtype=torch.bfloat16).cuda() for t in (1, 70))

    def step(q, new):
        cache.append(new, new)
        return cache.attend(q)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(small, new_small), step(large, new_large)
    torch.cuda.current_stream().wait_stream(stream)
    graphs, results = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, q, new in zip(graphs, (small, large), (new_small, new_large)):
        with torch.cuda.graph(graph):
            results.append(step(q, new))
    for n in range(3):
        for graph, result, q, new in zip(graphs, results, (small, large), (new_small, new_large)):
            graph.replay()
            got = [x.clone() for x in result]
            want = step(q, new)
            ops.check_status("cuda:0")
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        table.advance(3)


def test_nothing_to_do():
    cache = over(*(torch.zeros(4, 1, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)),
                 torch.zeros(1, 4, dtype=torch.int32, device="cuda"), [0], 16)
    none = torch.zeros(1, 0, 1, 64, dtype=torch.bfloat16, device="cuda")
    assert cache.append(none, none) is None
    out, lse = cache.attend(none)
    assert out.shape == (1, 0, 1, 64) and lse.shape == (1, 0, 1)
    cache.keep(torch.zeros(1, 0, dtype=torch.int32, device="cuda"))
    mask, depth = ops.tree_mask(torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert mask.shape == (0, 0) and depth.shape == (0,)
    ops.check_status("cuda:0")


def test_refusals_on_the_gpu():
    cache = over(*(torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)),
                 torch.zeros(2, 2, dtype=torch.int32, device="cuda"), [0, 0], 16)
    x = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16, device="cuda")
    for call, word in ((lambda: cache.attend(x.half()), "bfloat16"), (lambda: cache.attend(x[:1]), "must be"), (lambda: cache.attend(x[:, :, :1]), "heads"),
                       (lambda: cache.attend(x, counts=[1, 2]), "counts"), (lambda: cache.attend(x, counts=torch.ones(2, device="cuda")), "counts"),
                       (lambda: cache.attend(x, tree=torch.zeros(3, 2, dtype=torch.int32, device="cuda")), "tree"),
                       (lambda: cache.attend(x, tree=torch.zeros(3, 1, dtype=torch.int32)), "tree"),
                       (lambda: cache.attend(x, status=torch.zeros(1, device="cuda")), "status"),
                       (lambda: cache.append(x, x[:, :2]), "share"), (lambda: cache.append(x, x, x), "rotation"),
                       (lambda: cache.append(x, x.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"),
                       (lambda: cache.keep(torch.zeros(2, dtype=torch.int32, device="cuda")), "path"),
                       (lambda: cache.keep(torch.zeros(2, 1, dtype=torch.int32)), "path"),
                       (lambda: cache.keep(torch.zeros(3, 1, dtype=torch.int32, device="cuda")), "path"),
                       (lambda: ops.tree_mask(torch.zeros(1, 2, 3, dtype=torch.int32, device="cuda")), "parents")):
        with pytest.raises(ValueError, match=word):
            call()
    with pytest.raises(RuntimeError):
        cache.attend(x.cpu())
