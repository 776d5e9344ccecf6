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
