"""The paged 16-bit cache on the GPU against its formulas in 64 bits: append, attention, accepted rows, tree masks."""
import math

import pytest
import torch

import block_reference
import page_reference as ref
from nanokv_b200 import ops, page_cache
from nanokv_b200.page_cache import PageCache, PageTable
from nanokv_b200.rotary import Rotary

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def made(batch, capacity, heads, dim, dtype, page, seed, lengths, garbage=math.nan):
    """A cache whose sequences hold random tokens up to their capacity, NaN in pages that are nobody's, and its arrays on the host."""
    table, pages = ref.scattered(batch, capacity, page, seed)
    k, v = (torch.full((pages, heads, page, dim), garbage, dtype=dtype) for _ in range(2))
    used = table.flatten().long()
    k[used] = ref.randn(len(used), heads, page, dim, seed=seed + 1, dtype=dtype) * torch.exp(0.5 * ref.randn(1, heads, 1, dim, seed=seed + 3)).to(dtype)
    v[used] = ref.randn(len(used), heads, page, dim, seed=seed + 2, dtype=dtype)
    pt = PageTable.over(table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), pages=pages, page=page)
    return PageCache.over(pt, k.cuda(), v.cuda()), k, v, table


def spoiled(cache, k, v, table, lengths, counts):
    """Everything behind a sequence's last pending token NaN, on both sides."""
    page = k.shape[2]
    for b, (n, c) in enumerate(zip(lengths, counts)):
        for t in range(n + c, table.shape[1] * page):
            k[int(table[b, t // page]), :, t % page] = math.nan
            v[int(table[b, t // page]), :, t % page] = math.nan
    cache.k_pages.copy_(k)
    cache.v_pages.copy_(v)


def check_attention(cache, k, v, table, q, lengths, *, counts=None, mask=None, tree=None, causal=True, scale=None, atol=0.0):
    """One call against the formula.  Bounds: the result's own rounding; weights rounded to 16 bits, and as much again for the
    running references, times the sum of p |v|; scores as fp32 sums of at most 128 products in any order, and exponentials of
    them (a relative 2^-18 of the sum of magnitudes); fp32 sums over n tokens; fp16 weights below 2^-14, which have half a
    step of 2^-25 each where the largest has at least 2^7."""
    B, T, H, D = q.shape
    n = [T] * B if counts is None else counts
    out, lse = cache.attend(q.cuda() if not q.is_cuda else q, counts=None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda(),
                            tree=tree, causal=causal, scale=scale)
    ops.check_status(out.device)
    if mask is None:
        mask = torch.ones(B, T, T, dtype=torch.bool)
        mask = mask.tril() if causal else mask
    want, want_lse, spread, size = ref.attention(q, k, v, table, lengths, n, mask, D ** -0.5 if scale is None else scale)
    unit = ref.UNIT[q.dtype]
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(torch.isnan(lse), torch.isnan(want_lse))
    ok = ~torch.isnan(want_lse)
    score = 2.0 ** -18 * size.clamp_min(1.0)
    seen = ok & (want_lse > -math.inf)
    assert torch.equal(lse[ok & ~seen], want_lse[ok & ~seen])
    assert not out[ok & ~seen].any()
    tokens = max(a + b for a, b in zip(lengths, n))
    assert not seen.any() or ((lse - want_lse).abs() <= score + 2.0 ** -22 * want_lse.abs() + 2.0 ** -23 * tokens)[seen].all()
    assert torch.isnan(out[~ok]).all()
    finite = want.isfinite() & ok[..., None]
    assert torch.equal(out.isfinite()[ok], finite[ok])
    bound = unit * want.abs() + (2 * unit + 4 * score[..., None] + 2.0 ** -22 * tokens) * spread + 1e-7 + atol
    if q.dtype == torch.float16:
        bound = bound + 2.0 ** -32 * tokens * float(v[v.isfinite()].abs().max())
    error = torch.where(finite, (out - want.nan_to_num()).abs() / bound, 0.0)
    assert (error <= 1).all(), float(error.max())


# ------------------------------------------------------------------ append
def appended(k_pages, v_pages, table, lengths, counts, k, v):
    for b, (n, c) in enumerate(zip(lengths, counts)):
        ref.put(k_pages, table, b, n, k[b, :c])
        ref.put(v_pages, table, b, n, v[b, :c])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rotary_dim,layout", [(64, 64, "half"), (64, 16, "interleaved"), (128, 128, "interleaved"), (128, 32, "half"), (128, 0, "half")])
@pytest.mark.parametrize("page,lengths,tokens,counts", [(16, [0, 31], 1, None), (16, [15, 16, 40], 33, [33, 0, 1]), (64, [63], 130, None),
                                                       (32, [5, 6], 7, [7, 3]), (128, [200, 0], 64, None)])
def test_append_writes_rotated_keys_values_and_queries(page, lengths, tokens, counts, dim, rotary_dim, layout, dtype):
    B, H, G = len(lengths), 2, 3
    cache, kp, vp, table = made(B, max(lengths) + tokens + page, H, dim, dtype, page, 3, lengths)
    qkv = ref.randn(B, tokens, H * (G + 2), dim, seed=9, dtype=dtype)
    q, k, v = qkv.cuda().split([H * G, H, H], 2)
    n = [tokens] * B if counts is None else counts
    given = None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()
    k_host, v_host = k.cpu(), v.cpu()
    if rotary_dim:
        rot = Rotary(dim, 512, rotary_dim=rotary_dim, layout=layout)
        positions = (torch.arange(tokens)[None] * 2 + torch.tensor(lengths)[:, None]).to(torch.int32)
        got_q = cache.append(k, v, q, counts=given, rotary=rot, positions=positions.cuda())
        # the same bits as the rotation on its own, which is held to the formula
        want_q, want_k = rot.apply(q, k, positions=positions.cuda())
        assert torch.equal(got_q, want_q) and got_q.is_contiguous()
        exact = block_reference.rotated(q.cpu(), rot.table.cpu(), positions, layout)
        assert ((got_q.double().cpu() - exact).abs() <= ref.UNIT[dtype] * exact.abs() + 2.0 ** -22 * q.cpu().double().abs().amax()).all()
        k_host = want_k.cpu()
    else:
        assert cache.append(k, v, counts=given) is None
    ops.check_status(k.device)
    appended(kp, vp, table, lengths, n, k_host, v_host)
    assert torch.equal(cache.k_pages.cpu().view(torch.int16), kp.view(torch.int16))
    assert torch.equal(cache.v_pages.cpu().view(torch.int16), vp.view(torch.int16))


@pytest.mark.parametrize("dtype", TYPES)
def test_append_by_default_turns_by_the_settled_lengths(dtype):
    lengths = [0, 77, 130]
    cache, *_ = made(3, 200, 2, 128, dtype, 64, 5, lengths)
    q, k, v = (ref.randn(3, 5, h, 128, seed=h, dtype=dtype).cuda() for h in (4, 2, 2))
    rot = Rotary(128, 200)
    got_q = cache.append(k, v, q, rotary=rot)
    first = cache.k_pages.clone()
    positions = (cache.table.lengths[:, None] + torch.arange(5, device="cuda")).to(torch.int32)
    want_q = cache.append(k, v, q, rotary=rot, positions=positions)
    assert torch.equal(got_q, want_q) and torch.equal(first.view(torch.int16), cache.k_pages.view(torch.int16))


@pytest.mark.parametrize("offset", [1, 3, 8])
def test_append_takes_rows_that_start_anywhere(offset):
    flat = ref.randn(2 * 3 * 2 * 128 + 16, seed=4, dtype=torch.bfloat16).cuda()
    x = flat[offset:offset + 2 * 3 * 2 * 128].view(2, 3, 2, 128)
    rot = Rotary(128, 64)
    results = []
    for rows in (x, x.clone()):
        cache, *_ = made(2, 64, 2, 128, torch.bfloat16, 16, 6, [9, 20], garbage=0.0)
        results.append((cache.append(rows, rows, rows, rotary=rot), cache.k_pages, cache.v_pages))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_positions_outside_the_table_are_nan():
    cache, *_ = made(1, 64, 1, 64, torch.bfloat16, 16, 6, [9], garbage=0.0)
    x = ref.randn(1, 3, 1, 64, seed=1, dtype=torch.bfloat16).cuda()
    q = cache.append(x, x, x, rotary=Rotary(64, 8), positions=torch.tensor([[7, 8, -1]], dtype=torch.int32).cuda())
    assert torch.isnan(q[0, :, 0]).any(-1).tolist() == [False, True, True]


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("group,tokens", [(1, 1), (5, 1), (4, 8), (3, 11), (5, 13), (4, 17), (8, 16), (43, 3), (4, 33), (1, 300), (16, 40)])
def test_causal_attention_over_lengths_at_borders(group, tokens, page, dim, dtype):
    lengths = [0, 1, 127, 128, 129, 300 if page == 16 else 1000]
    cache, k, v, table = made(len(lengths), max(lengths) + tokens, 2, dim, dtype, page, 21, lengths)
    spoiled(cache, k, v, table, lengths, [tokens] * len(lengths))
    q = ref.randn(len(lengths), tokens, 2 * group, dim, seed=22, dtype=dtype, std=1.5)
    check_attention(cache, k, v, table, q, lengths)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 64), (128, 16)])
@pytest.mark.parametrize("group,tokens,shared", [(1, 2, False), (2, 16, True), (5, 16, False), (4, 31, False), (4, 32, True), (1, 33, False), (4, 63, False),
                                                 (2, 150, True), (8, 65, False)])
def test_trees(group, tokens, shared, dim, page, dtype):
    lengths = [0, 3, 97, 128, 250]
    B = len(lengths)
    cache, k, v, table = made(B, max(lengths) + tokens, 2, dim, dtype, page, 31, lengths)
    parents = torch.stack([ref.tree(tokens, 40 + (0 if shared else b)) for b in range(B)])
    mask = torch.stack([ref.sees(p) for p in parents])
    counts = None if shared else [tokens, 1, max(0, tokens - 3), 0, tokens]
    spoiled(cache, k, v, table, lengths, [tokens] * B if counts is None else counts)
    bits, depth = ops.tree_mask((parents[0] if shared else parents).cuda())
    assert torch.equal(bits.cpu(), ref.packed(mask[0] if shared else mask))
    assert torch.equal(depth.cpu().long(), (mask[0] if shared else mask).sum(-1) - 1)
    q = ref.randn(B, tokens, 2 * group, dim, seed=32, dtype=dtype, std=1.5)
    check_attention(cache, k, v, table, q, lengths, counts=counts, mask=mask, tree=bits)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,tokens", [(1, 20), (4, 12), (2, 60), (8, 50)])
def test_any_mask_and_rows_that_see_nothing(group, tokens, dtype):
    """Bits that are no tree's, among them none at all over an empty sequence."""
    lengths = [0, 130, 0]
    cache, k, v, table = made(3, 130 + tokens, 1, 128, dtype, 64, 41, lengths)
    mask = torch.rand(3, tokens, tokens, generator=torch.Generator().manual_seed(1)) < 0.2
    mask[:, ::3] = False
    spoiled(cache, k, v, table, lengths, [tokens] * 3)
    q = ref.randn(3, tokens, group, 128, seed=42, dtype=dtype)
    check_attention(cache, k, v, table, q, lengths, mask=mask, tree=ref.packed(mask).cuda())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,tokens", [(1, 1), (4, 20), (1, 400)])
def test_all_pending_tokens_visible_and_counts(group, tokens, dtype):
    lengths, counts = [100, 0, 333, 128], [tokens, tokens // 2, 0, max(1, tokens - 1)]
    cache, k, v, table = made(4, 333 + tokens, 3, 64, dtype, 32, 51, lengths)
    spoiled(cache, k, v, table, lengths, counts)
    q = ref.randn(4, tokens, 3 * group, 64, seed=52, dtype=dtype)
    check_attention(cache, k, v, table, q, lengths, counts=counts, causal=False)


@pytest.mark.parametrize("group,tokens", [(1, 3), (3, 16), (4, 30), (8, 40), (1, 200)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_a_query_does_not_see_has_no_part(bad, dtype, group, tokens):
    """Keys and values of masked pending tokens that are not finite; rows that see such a value get it."""
    lengths = [0, 126, 200]
    cache, k, v, table = made(3, 200 + tokens, 1, 128, dtype, 16, 61, lengths)
    mask = torch.stack([ref.sees(ref.tree(tokens, 70 + b)) for b in range(3)])
    spoiled(cache, k, v, table, lengths, [tokens] * 3)
    node = tokens - 2
    for b, n in enumerate(lengths):
        ref.put(v, table, b, n + node, torch.full((1, 1, 128), bad))
        ref.put(k, table, b, n + tokens - 1, torch.full((1, 1, 128), bad))
        mask[b, node + 1] = False              # nobody but the last query sees the last token, and it not the one before
        mask[b, node + 1, node + 1] = True
    cache.k_pages.copy_(k)
    cache.v_pages.copy_(v)
    q = ref.randn(3, tokens, group, 128, seed=62, dtype=dtype)
    check_attention(cache, k, v, table, q[:, :, :], lengths, mask=mask, tree=ref.packed(mask).cuda()) if not math.isinf(bad) else \
        check_rows(cache, k, v, table, q, lengths, mask, tokens - 1)


def check_rows(cache, k, v, table, q, lengths, mask, rows):
    """As ``check_attention`` for the first ``rows`` queries: an infinite key's product with the last one has no sign to tell."""
    out, lse = cache.attend(q.cuda(), tree=ref.packed(mask).cuda())
    ops.check_status(out.device)
    want, want_lse, spread, size = ref.attention(q, k, v, table, lengths, [q.shape[1]] * 3, mask, q.shape[3] ** -0.5)
    out, lse, want, want_lse, spread, size = (x[:, :rows] for x in (out.double().cpu(), lse.double().cpu(), want, want_lse, spread, size))
    unit = ref.UNIT[q.dtype]
    score = 2.0 ** -18 * size.clamp_min(1.0)
    assert ((lse - want_lse).abs() <= score + 2.0 ** -14).all()
    assert torch.equal(out.isfinite(), want.isfinite())
    finite = want.isfinite()
    assert torch.equal(out[~finite].nan_to_num(), want[~finite].nan_to_num())
    bound = unit * want.abs() + (2 * unit + 4 * score[..., None] + 2.0 ** -13) * spread + 1e-6
    assert ((out - want).abs() <= bound)[finite].all()


@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0])
def test_scales(scale):
    lengths = [50, 200]
    cache, k, v, table = made(2, 220, 2, 128, torch.bfloat16, 64, 71, lengths)
    q = ref.randn(2, 6, 8, 128, seed=72, dtype=torch.bfloat16)
    check_attention(cache, k, v, table, q, lengths, scale=scale)
    with pytest.raises(ValueError, match="finite"):
        cache.attend(q.cuda(), scale=math.inf)


@pytest.mark.parametrize("rows", [1, 40, 100, 200])
def test_values_from_the_smallest_to_the_largest(rows):
    """bf16 values up to its largest, in a sum that never passes it; scores that rise by hundreds along a sequence."""
    n = 700
    cache, k, v, table = made(1, n + rows, 1, 64, torch.bfloat16, 64, 81, [n])
    v = torch.where(v.isfinite(), v.sign() * 3e38 * (v.float().abs() / 8).clamp(0, 1), v.float()).to(torch.bfloat16)
    cache.v_pages.copy_(v)
    q = ref.randn(1, rows, 1, 64, seed=82, dtype=torch.bfloat16)
    check_attention(cache, k, v, table, q, [n])
    for i in range(n):
        ref.put(k, table, 0, i, torch.full((1, 1, 64), i / 4.0))
    cache.k_pages.copy_(k)
    check_attention(cache, k, v, table, torch.ones(1, rows, 1, 64, dtype=torch.bfloat16), [n])
    check_attention(cache, k, v, table, -torch.ones(1, rows, 1, 64, dtype=torch.bfloat16), [n])


@pytest.mark.parametrize("group,tokens", [(1, 1), (4, 40)])
def test_scores_of_minus_infinity_leave_a_row_empty(group, tokens):
    cache, k, v, table = made(1, 100 + tokens, 1, 64, torch.bfloat16, 64, 91, [100])
    k[table.flatten().long()] = -math.inf
    cache.k_pages.copy_(k)
    out, lse = cache.attend(torch.ones(1, tokens, group, 64, dtype=torch.bfloat16, device="cuda"))
    assert not out.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("tokens,offset", [(1, 0), (1, 1), (40, 3), (200, 1)])
def test_queries_with_strides_of_their_own(tokens, offset):
    lengths = [90, 130]
    cache, k, v, table = made(2, 400, 2, 128, torch.float16, 32, 101, lengths)
    flat = ref.randn(2 * tokens * 9 * 128 + 8, seed=102, dtype=torch.float16).cuda()
    q = flat[offset:offset + 2 * tokens * 9 * 128].view(2, 9, tokens, 128).transpose(1, 2)[:, :, 1:7]
    check_attention(cache, k, v, table, q, lengths)


def test_batches_of_more_sequences_than_one_launch_takes():
    lengths = [(37 * i) % 150 for i in range(230)]
    cache, k, v, table = made(230, 160, 1, 64, torch.bfloat16, 16, 111, lengths)
    counts = [i % 4 for i in range(230)]
    spoiled(cache, k, v, table, lengths, counts)
    q = ref.randn(230, 3, 2, 64, seed=112, dtype=torch.bfloat16)
    check_attention(cache, k, v, table, q, lengths, counts=counts)


@pytest.mark.parametrize("heads,tokens,length", [(1, 1, 70001), (3, 5, 20000), (2, 129, 9000)])
def test_long_sequences_are_cut_and_joined(heads, tokens, length):
    cache, k, v, table = made(1, length + tokens, heads, 64, torch.bfloat16, 128, 121, [length])
    q = ref.randn(1, tokens, heads, 64, seed=122, dtype=torch.bfloat16)
    check_attention(cache, k, v, table, q, [length])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group,tokens", [(128, 8, 1), (64, 4, 10), (128, 5, 16), (128, 2, 90)])
def test_thread_blocks_with_many_pieces_of_many_tiles(dim, group, tokens, dtype):
    """Rings that go round several times within a piece, and several pieces a thread block, with masked tiles at their ends."""
    heads = 16
    lengths = [2138 - 61 * i for i in range(31)]
    counts = [0 if i % 8 == 5 else max(1, tokens - i % 3) for i in range(31)]
    cache, k, v, table = made(31, 2138 + tokens, heads, dim, dtype, 64, 125, lengths)
    spoiled(cache, k, v, table, lengths, counts)
    q = ref.randn(31, tokens, heads * group, dim, seed=126, dtype=dtype).cuda()
    # sequences and heads apart from one another; one of them against the formula
    out, lse = cache.attend(q, counts=torch.tensor(counts, dtype=torch.int32).cuda())
    ops.check_status(out.device)
    pages = torch.cat([table, table], 0).cuda()
    for b in (0, 1, 5, 17, 30):
        one = PageTable.over(pages[b:b + 1].contiguous(), torch.tensor([lengths[b]], dtype=torch.int32).cuda(), pages=cache.table.pages, page=64)
        for h in (0, 7, 15):
            part = PageCache.over(one, cache.k_pages[:, h:h + 1].contiguous(), cache.v_pages[:, h:h + 1].contiguous())
            rows = q[b:b + 1, :, h * group:(h + 1) * group]
            check_attention(part, k[:, h:h + 1], v[:, h:h + 1], table[b:b + 1], rows, [lengths[b]], counts=[counts[b]])
            alone, lse_alone = part.attend(rows, counts=torch.tensor([counts[b]], dtype=torch.int32).cuda())
            got, lse_got = out[b:b + 1, :, h * group:(h + 1) * group], lse[b:b + 1, :, h * group:(h + 1) * group]
            seen = lse_alone > -math.inf
            assert torch.equal(seen, lse_got > -math.inf)
            assert not seen.any() or ((lse_alone - lse_got).abs()[seen] <= 2.0 ** -12).all()
            # both are within the bounds of check_attention of the formula, where values are a few units at most
            assert ((alone.float() - got.float()).abs() <= 6 * ref.UNIT[dtype] * 6).all()


def test_results_are_the_same_every_time():
    lengths = [500, 1, 900]
    cache, k, v, table = made(3, 1000, 2, 128, torch.bfloat16, 64, 131, lengths)
    for tokens, group in ((1, 4), (20, 4), (50, 4)):
        q = ref.randn(3, tokens, 2 * group, 128, seed=132, dtype=torch.bfloat16).cuda()
        out, lse = cache.attend(q)
        for _ in range(3):
            again, lse_again = cache.attend(q)
            assert torch.equal(out, again) and torch.equal(lse, lse_again)


def test_the_formula_kernel_agrees():
    """The kernel that computes the formula on CUDA cores, where the tensor cores are switched off."""
    lengths = [0, 100, 129]
    cache, k, v, table = made(3, 200, 2, 128, torch.bfloat16, 16, 141, lengths)
    mask = torch.stack([ref.sees(ref.tree(20, b)) for b in range(3)])
    spoiled(cache, k, v, table, lengths, [20] * 3)
    q = ref.randn(3, 20, 6, 128, seed=142, dtype=torch.bfloat16)
    ops.force_simt(True)
    try:
        check_attention(cache, k, v, table, q, lengths, mask=mask, tree=ref.packed(mask).cuda())
        check_attention(cache, k, v, table, q, lengths, counts=[20, 0, 7])
        check_attention(cache, k, v, table, q, lengths, causal=False)
    finally:
        ops.force_simt(False)


# ------------------------------------------------------------------ accepted rows
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,page", [(64, 1, 16), (128, 8, 64), (128, 40, 32)])
def test_keep_moves_the_path_to_the_front(dim, heads, page, dtype):
    lengths, tokens = [0, 13, 62, 127], 40
    caches, hosts = [], []
    table = None
    for layer in range(3):
        cache, k, v, table = made(4, 200, heads, dim, dtype, page, 151, lengths)
        k, v = k + layer, v + layer
        caches.append(PageCache.over(caches[0].table if caches else cache.table, k.cuda(), v.cuda()))
        hosts.append((k, v))
    path = torch.stack([torch.randperm(tokens, generator=torch.Generator().manual_seed(b))[:20].sort()[0] for b in range(4)]).to(torch.int32)
    path[1] = torch.arange(20)
    path[2] = torch.arange(20) + 1
    counts = [20, 20, 17, 0]
    page_cache.keep(caches, path.cuda(), torch.tensor(counts, dtype=torch.int32).cuda())
    ops.check_status("cuda:0")
    for cache, (k, v) in zip(caches, hosts):
        for got, pool in ((cache.k_pages, k), (cache.v_pages, v)):
            want = pool.clone()
            for b, (n, c) in enumerate(zip(lengths, counts)):
                held = ref.rows_of(pool, table, b, n + tokens)
                ref.put(want, table, b, n, held[n + path[b, :c].long()])
            assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
    before = [c.k_pages.clone() for c in caches]
    caches[1].keep(path[:, :1].cuda())          # one cache, all of a path of one
    assert torch.equal(before[0].view(torch.int16), caches[0].k_pages.view(torch.int16))


def test_more_caches_than_one_launch_takes():
    cache, k, v, table = made(1, 64, 1, 64, torch.bfloat16, 16, 161, [5], garbage=0.0)
    pools = [(torch.stack([k + i for i in range(70)]).cuda(), torch.stack([v - i for i in range(70)]).cuda())]
    caches = [PageCache.over(cache.table, pools[0][0][i], pools[0][1][i]) for i in range(70)]
    page_cache.keep(caches, torch.tensor([[2, 9]], dtype=torch.int32).cuda())
    for i in (0, 63, 64, 69):
        for pool, host in ((pools[0][0][i], k + i), (pools[0][1][i], v - i)):
            assert torch.equal(ref.rows_of(pool.cpu(), table, 0, 7)[5:], ref.rows_of(host, table, 0, 15)[[7, 14]])


# ------------------------------------------------------------------ tree masks
@pytest.mark.parametrize("batch,tokens", [(1, 1), (3, 31), (2, 32), (5, 33), (1, 64), (2, 511), (1, 4096)])
def test_tree_masks(batch, tokens):
    parents = torch.stack([ref.tree(tokens, 7 * b + tokens) for b in range(batch)])
    if batch > 1:
        parents[0] = ref.chain(tokens)
        parents[1] = -1
    mask, depth = ops.tree_mask(parents.cuda())
    ops.check_status("cuda:0")
    want = torch.stack([ref.sees(p) for p in parents])
    assert torch.equal(mask.cpu(), ref.packed(want)) and torch.equal(depth.cpu().long(), want.sum(-1) - 1)


def test_parents_that_do_not_come_first_count_as_none():
    parents = torch.tensor([0, 5, -2, 2 ** 31 - 1, 2], dtype=torch.int32)
    mask, depth = ops.tree_mask(parents.cuda())
    with pytest.raises(RuntimeError, match="parent"):
        ops.check_status("cuda:0")
    assert mask.flatten().tolist() == [1, 2, 4, 8, 4 | 16] and depth.tolist() == [0, 0, 0, 0, 1]


# ------------------------------------------------------------------ as they are used together
@pytest.mark.parametrize("captured", [False, True])
def test_a_draft_verified_and_settled_step_by_step(captured):
    """Prompt, then drafts: rotate and store, attend as a tree, keep the accepted branch, settle it; the cache then holds what a
    chain of the accepted tokens holds.  Captured once, the step is replayed while the sequences grow."""
    B, H, G, D, T, steps, dtype = 2, 2, 2, 64, 7, 4, torch.bfloat16
    parents = torch.tensor([-1, -1, 0, 0, 1, 2, 5], dtype=torch.int32)
    mask = ref.sees(parents)
    paths = torch.tensor([[0, 2, 5, 6], [1, 4, 4, 4]], dtype=torch.int32)
    counts = [4, 2]
    rot = Rotary(D, 256)
    table = PageTable(B, 256, pages=40, page=16)
    table.reserve([100, 90])
    caches = [PageCache(table, H, D, dtype=dtype) for _ in range(2)]
    chain_k = [[[] for _ in range(B)] for _ in caches]
    chain_v = [[[] for _ in range(B)] for _ in caches]
    prompt = [ref.randn(B, 20, H * (G + 2), D, seed=i, dtype=dtype) for i in range(2)]
    for i, cache in enumerate(caches):
        q, k, v = prompt[i].cuda().split([H * G, H, H], 2)
        cache.append(k, v, q, rotary=rot)
        at = torch.arange(20, dtype=torch.int32).expand(B, 20).contiguous()
        turned = rot.apply(k, positions=at.cuda()).cpu()
        for b in range(B):
            chain_k[i][b].append(turned[b])
            chain_v[i][b].append(v[b].cpu())
    table.advance(20)
    lengths = [20, 20]
    bits, depth = ops.tree_mask(parents.cuda())
    rows = torch.zeros(2, B, T, H * (G + 2), D, dtype=dtype, device="cuda")
    accepted = torch.tensor(counts, dtype=torch.int32).cuda()
    path = paths.cuda()
    results = []

    def step():
        positions = table.lengths[:, None] + depth
        results.clear()
        for i, cache in enumerate(caches):
            q, k, v = rows[i].split([H * G, H, H], 2)
            turned = cache.append(k, v, q, rotary=rot, positions=positions)
            results.append((turned, *cache.attend(turned, tree=bits)))
        page_cache.keep(caches, path, accepted)
        table.advance(accepted)

    graph = None
    if captured:
        stream = torch.cuda.Stream()
        before = table.lengths.clone(), [(c.k_pages.clone(), c.v_pages.clone()) for c in caches]
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        table.lengths.copy_(before[0])
        for c, (k, v) in zip(caches, before[1]):
            c.k_pages.copy_(k)
            c.v_pages.copy_(v)
    for s in range(steps):
        fresh = ref.randn(2, B, T, H * (G + 2), D, seed=100 + s, dtype=dtype)
        rows.copy_(fresh)
        graph.replay() if captured else step()
        ops.check_status("cuda:0")
        assert table.lengths.tolist() == [n + c for n, c in zip(lengths, counts)]
        for i in range(2):
            k, v = fresh[i][:, :, H * G:H * G + H], fresh[i][:, :, H * G + H:]
            at = (torch.tensor(lengths)[:, None] + depth.cpu()).to(torch.int32)
            turned = rot.apply(k.contiguous().cuda(), positions=at.cuda()).cpu()
            # the attention of this step, over the chain and the draft
            flat = [torch.stack([torch.nn.functional.pad(torch.cat([*past[b], new[b]]), (0, 0, 0, 0, 0, 120 - sum(map(len, past[b])) - T))
                                 for b in range(B)]) for past, new in ((chain_k[i], turned), (chain_v[i], v))]
            own_table = torch.arange(B * 120, dtype=torch.int32).reshape(B, 120)
            pools = [x.reshape(B * 120, H, 1, D) for x in flat]
            turned_q, out, lse = results[i]
            want, want_lse, spread, size = ref.attention(turned_q, *pools, own_table, lengths, [T] * B, mask.expand(B, T, T), D ** -0.5)
            unit = ref.UNIT[dtype]
            score = 2.0 ** -18 * size.clamp_min(1.0)
            assert ((lse.double().cpu() - want_lse).abs() <= score + 2.0 ** -14).all()
            bound = unit * want.abs() + (2 * unit + 4 * score[..., None] + 2.0 ** -14) * spread + 1e-7
            assert ((out.double().cpu() - want).abs() <= bound).all()
            for b in range(B):
                nodes = paths[b, :counts[b]].long()
                chain_k[i][b].append(turned[b, nodes])
                chain_v[i][b].append(v[b, nodes])
        lengths = [n + c for n, c in zip(lengths, counts)]
    for i, cache in enumerate(caches):
        for b in range(B):
            for pool, past in ((cache.k_pages, chain_k[i][b]), (cache.v_pages, chain_v[i][b])):
                assert torch.equal(ref.rows_of(pool.cpu(), table.table.cpu(), b, lengths[b]), torch.cat(past))


def test_another_stream_than_the_tensors_own():
    lengths = [300, 40]
    cache, k, v, table = made(2, 400, 2, 64, torch.bfloat16, 64, 171, lengths)
    q = ref.randn(2, 4, 4, 64, seed=172, dtype=torch.bfloat16).cuda()
    want = cache.attend(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = cache.attend(q)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_calls_at_once():
    lengths = [3000, 40]
    cache, k, v, table = made(2, 3100, 2, 64, torch.bfloat16, 64, 181, lengths)
    q = ref.randn(2, 40, 4, 64, seed=182, dtype=torch.bfloat16).cuda()
    small = q[:, :1].contiguous()
    want, want_small = cache.attend(q), cache.attend(small)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(20):
        for s, x, r in zip(streams, (q, small), results):
            with torch.cuda.stream(s):
                r.append(cache.attend(x))
    torch.cuda.synchronize()
    for got in results[0]:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for got in results[1]:
        assert all(torch.equal(a, b) for a, b in zip(got, want_small))


# ------------------------------------------------------------------ pages and lengths that cannot be followed
def test_tokens_without_a_page_are_reported_and_left_out():
    cache, k, v, table = made(2, 64, 1, 64, torch.bfloat16, 16, 191, [30, 2], garbage=0.0)
    cache.table.table[0, 2] = -1                       # tokens 32 .. 47 of the first sequence
    cache.table.table[1, 0] = cache.table.pages        # and the first sixteen of the second
    before_k = cache.k_pages.clone()
    x = torch.ones(2, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    cache.append(x, x)
    with pytest.raises(RuntimeError, match="without a page"):
        ops.check_status("cuda:0")
    changed = (cache.k_pages != before_k).any(-1).sum()
    assert changed == 2                                # tokens 30 and 31
    out, lse = cache.attend(x)
    with pytest.raises(RuntimeError, match="without a page"):
        ops.check_status("cuda:0")
    assert not torch.isnan(out).any()
    cache.keep(torch.tensor([[1, 3], [0, 1]], dtype=torch.int32).cuda())
    with pytest.raises(RuntimeError, match="without a page"):
        ops.check_status("cuda:0")


@pytest.mark.parametrize("lengths,counts", [([-5, 63], None), ([2 ** 31 - 1, 10], None), ([64, 64], [4, 1]), ([3, 3], [-1, 2 ** 31 - 1])])
def test_lengths_and_counts_out_of_range_are_reported(lengths, counts):
    cache, *_ = made(2, 64, 1, 64, torch.bfloat16, 16, 201, lengths, garbage=0.0)
    given = None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()
    x = torch.ones(2, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: cache.append(x, x, counts=given), lambda: cache.attend(x, counts=given),
                 lambda: cache.attend(x, counts=given, tree=torch.full((4, 1), -1, dtype=torch.int32, device="cuda"))):
        call()
        with pytest.raises(RuntimeError, match="out of range"):
            ops.check_status("cuda:0")


@pytest.mark.parametrize("path", [[0, 0], [2, 1], [-1, 2], [5, 2 ** 31 - 1]])
def test_paths_out_of_order_are_reported(path):
    cache, *_ = made(1, 64, 1, 64, torch.bfloat16, 16, 211, [50], garbage=0.0)
    cache.keep(torch.tensor([path], dtype=torch.int32).cuda())
    with pytest.raises(RuntimeError, match="path out of range"):
        ops.check_status("cuda:0")


def test_pools_of_more_than_32_bits_of_elements():
    """The last pages of a pool of 2^32 elements."""
    page, heads, D = 128, 8, 128
    pages = 2 ** 32 // (page * heads * D) + 2
    k, v = (torch.zeros(pages, heads, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    pt = PageTable.over(table, torch.tensor([0], dtype=torch.int32, device="cuda"), pages=pages, page=page)
    cache = PageCache.over(pt, k, v)
    new = [ref.randn(1, 300, heads, D, seed=s, dtype=torch.bfloat16).cuda() for s in (1, 2)]
    cache.append(*new)
    ops.check_status("cuda:0")
    for pool, x in ((k, new[0]), (v, new[1])):
        got = torch.cat([pool[pages - 1], pool[0], pool[pages - 2]], 1).transpose(0, 1)[:300]
        assert torch.equal(got, x[0])
    pt.advance(298)
    small = [torch.stack([pool[i].cpu() for i in (pages - 1, 0, pages - 2)]) for pool in (k, v)]
    own = torch.arange(3, dtype=torch.int32)[None]
    q = ref.randn(1, 2, heads * 2, D, seed=3, dtype=torch.bfloat16)
    check_attention(cache, *small, own, q, [298])
    cache.keep(torch.tensor([[1]], dtype=torch.int32, device="cuda"))
    assert torch.equal(k[pages - 2, :, 298 - 256], new[0][0, 299])
