"""What the paged cache's attention makes of its 16-bit weights: sums, means, single values that count."""
import math

import pytest
import torch

import page_reference as ref
from nanokv_b200 import ops
from nanokv_b200.page_cache import PageCache, PageTable

pytestmark = pytest.mark.gpu
# query heads of a kv head x tokens: four copies of the rows, one copy, units of 256 rows
ROWS = [(1, 1), (4, 8), (5, 13), (1, 100), (8, 16), (3, 43), (4, 150)]


def filled(keys, values, page, batch=1):
    """Sequences that all hold keys, values [tokens, kv_heads, D], in pages of their own."""
    tokens, heads, D = keys.shape
    entries = -(-tokens // page)
    table = torch.randperm(batch * entries, generator=torch.Generator().manual_seed(1)).reshape(batch, entries).to(torch.int32)
    pools = []
    for rows in (keys, values):
        padded = torch.nn.functional.pad(rows, (0, 0, 0, 0, 0, entries * page - tokens))
        pool = torch.empty(batch * entries, heads, page, D, dtype=rows.dtype)
        pool[table.long()] = padded.reshape(entries, page, heads, D).transpose(1, 2)
        pools.append(pool.cuda())
    return pools[0], pools[1], table.cuda()


def over(k, v, table, lengths, page):
    lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return PageCache.over(PageTable.over(table, lengths, pages=k.shape[0], page=page), k, v)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("length,batch", [(700, 1), (700, 40), (5000, 1)])
@pytest.mark.parametrize("group,tokens", ROWS)
def test_a_mean_of_one_value_is_that_value(group, tokens, length, batch, D):
    """A sink and otherwise equal scores, values that are the same for all tokens: every weight loses the same bits, and the mean must not.
    Each kv head has a sink of another height, so that the equal weights fall all over the range between two powers of two.  What is left are
    fp32 sums of up to 5,200 terms and, of up to 32 rows, weights of 2^-15: below 2^-11 together.  Half a step of a bf16 number is at least
    2^-10 of it (towards the smaller ones, from a power of two): the result is the value itself."""
    heads, page, dtype = 8, 64, torch.bfloat16
    keys = torch.full((length + tokens, heads, D), 0.125)
    keys[0] = 0.125 + torch.arange(1, heads + 1)[:, None] * 0.03125
    values = ref.randn(1, heads, D, seed=3, dtype=dtype).expand(length + tokens, heads, D)
    cache = over(*filled(keys.to(dtype), values, page, batch), [length] * batch, page)
    q = torch.ones(batch, tokens, heads * group, D, dtype=dtype, device="cuda")
    out, lse = cache.attend(q)
    ops.check_status("cuda:0")
    want = values[0].cuda().repeat_interleave(group, 0)
    assert torch.equal(out, want.expand_as(out))
    # lse: scores are exact (sums of equal numbers of a few bits, times a power of two or D ** -0.5 rounded to fp32)
    scale = float(torch.tensor(D ** -0.5, dtype=torch.float32))
    sink, other = keys[0, :, 0].to(dtype).double() * D * scale, 0.125 * D * scale
    seen = length + torch.arange(1, tokens + 1, dtype=torch.float64)
    total = other + torch.log(torch.exp(sink - other) + (seen[:, None] - 1))        # [tokens, heads]
    assert ((lse.double().cpu() - total.repeat_interleave(group, 1)).abs() <= 2.0 ** -16).all()


@pytest.mark.parametrize("group,tokens", ROWS)
def test_results_are_off_in_both_directions_alike(group, tokens):
    """Positive values: the mean of the relative errors is that of independent roundings.  Each is at most 2^-8 in size for the result's
    rounding and 2^-7 of it for the weights'; the mean of n of them stays below 6 * 2^-7 / sqrt(n) where they are independent (weights
    of a row are shared by its columns: n counts rows)."""
    length, heads, batch, D, dtype = 900, 4, 24, 128, torch.bfloat16
    keys = ref.randn(length + tokens, heads, D, seed=1, dtype=dtype)
    values = (1 + ref.randn(length + tokens, heads, D, seed=2).abs()).to(dtype)
    k, v, table = filled(keys, values, 32, batch)
    cache = over(k, v, table, [length] * batch, 32)
    q = ref.randn(batch, tokens, heads * group, D, seed=4, dtype=dtype).cuda()
    out, _ = cache.attend(q, causal=False)
    ops.check_status("cuda:0")
    rows = q.reshape(batch * tokens, heads, group, D).permute(1, 0, 2, 3).reshape(heads, -1, D).double()
    s = rows @ keys.cuda().double().permute(1, 2, 0) * D ** -0.5
    want = (torch.softmax(s, -1) @ values.cuda().double().transpose(0, 1)).reshape(heads, batch * tokens, group, D)
    want = want.permute(1, 0, 2, 3).reshape(batch, tokens, heads * group, D)
    error = (out.double() - want) / want
    assert error.abs().max() <= 2.0 ** -8 + 2.0 ** -7
    assert abs(float(error.mean())) <= 6 * 2.0 ** -7 / math.sqrt(batch * tokens * heads * group)


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("length", [0, 2, 9, 130, 1000])
@pytest.mark.parametrize("group,tokens", [(1, 1), (8, 1), (4, 3), (1, 32), (2, 16)])
def test_few_rows_keep_sixteen_bits_of_a_weight(group, tokens, length, D, page):
    """Up to 32 bf16 rows a kv head: a weight goes as two numbers that leave less than 2^-15 of it, so 2^-14 of the sum of p |v| covers
    that and the fp32 sums beside the scores' own error; without the second number it would be up to 2^-7."""
    heads, dtype, batch = 3, torch.bfloat16, 2
    lengths = [length, max(0, length - 1)]
    keys, values = (ref.randn(length + tokens, heads, D, seed=s, dtype=dtype) for s in (1, 2))
    k, v, table = filled(keys, values, page, batch)
    cache = over(k, v, table, lengths, page)
    q = ref.randn(batch, tokens, heads * group, D, seed=4, dtype=dtype)
    out, lse = cache.attend(q.cuda())
    ops.check_status("cuda:0")
    mask = torch.ones(batch, tokens, tokens, dtype=torch.bool).tril()
    want, want_lse, spread, size = ref.attention(q, k.cpu(), v.cpu(), table.cpu(), lengths, [tokens] * batch, mask, D ** -0.5)
    score = 2.0 ** -18 * size.clamp_min(1.0)          # fp32 sums of up to 128 products in any order, and their exponential
    # the result is rounded where it stands: half a step of it, a little more where the error takes it past a power of two
    bound = ref.UNIT[dtype] * want.abs() * (1 + 2.0 ** -7) + (2.0 ** -14 + 4 * score[..., None]) * spread + 1e-7
    assert ((out.double().cpu() - want).abs() <= bound).all()
    assert ((lse.double().cpu() - want_lse).abs() <= score + 2.0 ** -16).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,group,tokens", [(128, 8, 1), (64, 4, 10), (128, 5, 16), (128, 2, 90), (64, 3, 90)])
def test_every_tile_of_many_pieces_counts(dim, group, tokens, dtype):
    """31 sequences x 16 kv heads at once, rings that go round within a piece: results of single sequences and heads against the formula.
    Weights and result are off by their roundings, relative to the sum of p |v|, which for tokens of about equal weight is far below
    what one tile of 128 tokens in 2,138 adds to the mean."""
    heads, page = 16, 64
    lengths = [2138 - 61 * i for i in range(31)]
    counts = [0 if i % 8 == 5 else max(1, tokens - i % 3) for i in range(31)]
    table, pages = ref.scattered(31, 2138 + tokens, page, 5)
    gen = torch.Generator(device="cuda").manual_seed(6)
    k, v = (torch.randn(pages, heads, page, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    cache = over(k, v, table.cuda(), lengths, page)
    q = torch.randn(31, tokens, heads * group, dim, generator=gen, device="cuda").to(dtype)
    out, lse = cache.attend(q, counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
    ops.check_status("cuda:0")
    unit = ref.UNIT[dtype]
    for b in (0, 1, 5, 12, 17, 24, 30):
        for h in (0, 3, 7, 11, 15):
            part = slice(h * group, (h + 1) * group)
            mask = torch.ones(1, tokens, tokens, dtype=torch.bool).tril()
            want, want_lse, spread, size = ref.attention(q[b:b + 1, :, part], k[:, h:h + 1].cpu(), v[:, h:h + 1].cpu(), table[b:b + 1], lengths[b:b + 1],
                                                         counts[b:b + 1], mask, dim ** -0.5)
            got, got_lse = out[b:b + 1, :, part].double().cpu(), lse[b:b + 1, :, part].double().cpu()
            score = 2.0 ** -18 * size.clamp_min(1.0)
            seen = want_lse > -math.inf
            assert torch.equal(got_lse > -math.inf, seen) and not got[~seen].any()
            if not seen.any():
                continue
            assert ((got_lse - want_lse).abs() <= score + 2.0 ** -14)[seen].all()
            bound = unit * want.abs() + (2 * unit + 4 * score[..., None] + 2.0 ** -12) * spread + 1e-7
            if dtype == torch.float16:
                bound = bound + 2.0 ** -32 * 2300 * float(v.abs().max())
            assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("dtype,D,heads,tokens,length", [(torch.bfloat16, 128, 8, 2300, 33000), (torch.float16, 64, 8, 2000, 42000)])
def test_values_that_are_not_finite_in_units_that_are_cut(dtype, D, heads, tokens, length, bad):
    """Keys and values of more than 64 MB, several runs a thread block: a value of a pending token counts for the queries from it on."""
    page, total = 128, length + tokens
    gen = torch.Generator(device="cuda").manual_seed(1)
    pages = -(-total // page)
    k, v = (torch.randn(pages, heads, page, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)[None].contiguous()
    q = torch.randn(1, tokens, heads, D, generator=gen, device="cuda").to(dtype)
    cache = over(k, v, table, [length], page)
    want, want_lse = cache.attend(q)
    columns = [0, D // 2 - 1, D // 2, D - 1]
    first = {h: tokens * (h + 1) // (heads + 1) for h in range(heads)}      # the pending token of each head
    for h, t in first.items():
        entry, row = divmod(length + t, page)
        v[int(table[0, entry]), h, row, columns[h % 4]] = bad
    out, lse = cache.attend(q)
    ops.check_status("cuda:0")
    assert torch.equal(lse, want_lse)                                       # (values have no part in it)
    for h, t in first.items():
        hit = torch.zeros(tokens, D, dtype=torch.bool, device="cuda")
        hit[t:, columns[h % 4]] = True
        assert torch.equal(out[0, :, h].isfinite(), ~hit)
        # rows before it: the value, taken out, is not part of their sums
        assert torch.equal(out[0, :, h][~hit], want[0, :, h][~hit])
