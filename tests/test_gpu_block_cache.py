"""The 8-bit block cache on the GPU against its formulas in 64 bits: what is held, attention, eviction."""
import math
import random

import pytest
import torch

import block_reference as ref
from nanokv_b200 import ops
from nanokv_b200.block_cache import BLOCK, BlockCache
from nanokv_b200.rotary import Rotary

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def randn(*shape, seed, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def shuffled(cache, seed):
    """The cache with its slots in another order, as evictions leave them."""
    gen = torch.Generator().manual_seed(seed)
    cache.table.copy_(torch.rand(cache.table.shape, generator=gen).argsort(-1).to(torch.int32))
    return cache


def filled(lengths, heads, dim, dtype, seed, capacity=None, std_v=1.0):
    """A cache of sequences of these lengths, and the values it should hold."""
    n = max(max(lengths), 1)
    k = randn(len(lengths), n, heads, dim, seed=seed, dtype=dtype) * torch.exp(0.5 * randn(1, 1, heads, dim, seed=seed + 1)).to(dtype)
    v = randn(len(lengths), n, heads, dim, seed=seed + 2, dtype=dtype, std=std_v)
    cache = shuffled(BlockCache(len(lengths), heads, dim, capacity or n + 70, dtype=dtype), seed)
    cache.append(k.cuda(), v.cuda(), counts=lengths)
    return cache, *ref.held(k, v, lengths)


def check_attention(cache, hk, hv, q, *, counts=None, causal=True, scale=None, weights=True):
    """Results of one call against the formula.  Bounds: the result's own rounding; 16-bit weights in the product with V
    (their relative error times the sum of p |v|, and as much again for the running reference points); scores as fp32
    sums of at most 128 products (a relative 2^-18 of the sum of magnitudes leaves room for any order)."""
    B, T, H, D = q.shape
    q = q if q.is_cuda else q.cuda()
    given = torch.full_like(cache.weights, 0.25)
    out, lse = cache.attend(q, counts=counts, causal=causal, scale=scale, weights=given if weights else None)
    ops.check_status(q.device)
    n = [T] * B if counts is None else counts
    want, want_lse, spread, size, shares = ref.attention(q, hk, hv, cache.lengths, n, causal, D ** -0.5 if scale is None else scale)
    unit = ref.UNIT[q.dtype]
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(torch.isnan(lse), torch.isnan(want_lse))
    ok = ~torch.isnan(want_lse)
    score = 2.0 ** -18 * size.clamp_min(1.0)
    seen = ok & (want_lse > -math.inf)
    assert torch.equal(lse[ok & ~seen], want_lse[ok & ~seen])
    assert not seen.any() or ((lse - want_lse).abs() <= score + 2.0 ** -22 * want_lse.abs())[seen].all()
    assert not out[ok & ~seen].any()
    bound = unit * want.abs() + (2 * unit + 4 * score[..., None]) * spread + 1e-7
    assert ((out - want).abs() <= bound)[ok].all(), float(((out - want).abs() / bound)[ok].max())
    if weights and not torch.isnan(shares).any():
        got = given.double().cpu()
        full = torch.zeros_like(got)
        used = min(shares.shape[2], got.shape[2])
        full[:, :, :used] = shares[:, :, :used]
        worst = float(score.max())
        assert ((got - 0.25 - full).abs() <= 4 * worst * full + 2.0 ** -22).all()


# ------------------------------------------------------------------ what is held
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[0, 1], [63, 64], [65, 200], [129]])
def test_read_gives_what_the_formula_holds(lengths, dim, dtype):
    cache, hk, hv = filled(lengths, 3, dim, dtype, 11)
    k, v = cache.read(0, max(lengths))
    for got, want in ((k, hk), (v, hv)):
        # equal codes; the value is rounded to the type
        assert ((got.double().cpu() - want).abs() <= ref.UNIT[dtype] * want.abs() + 1e-30).all()
    a, b = max(0, max(lengths) - 70), max(lengths) + 1
    part_k, part_v = cache.read(a, b)
    assert torch.equal(part_k[:, :-1], k[:, a:]) and torch.equal(part_v[:, :-1], v[:, a:])
    assert not part_k[:, -1].any() and not part_v[:, -1].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_cache_does_not_depend_on_how_its_tokens_were_cut(dtype):
    k, v = (randn(2, 300, 2, 128, seed=s, dtype=dtype).cuda() for s in (1, 2))
    whole, cut = (BlockCache(2, 2, 128, 320, dtype=dtype) for _ in range(2))
    for cache in (whole, cut):
        for name in ("k_codes", "v_codes", "scales", "k_tail", "v_tail"):
            getattr(cache, name).zero_()
    whole.append(k, v)
    at, gen = 0, random.Random(5)
    while at < 300:
        n = min(300 - at, gen.choice([1, 1, 1, 7, 63, 64, 100]))
        cut.append(k[:, at:at + n], v[:, at:at + n])
        at += n
    assert cut.lengths == whole.lengths == [300, 300]
    for name in ("k_codes", "v_codes", "scales"):
        assert torch.equal(getattr(whole, name), getattr(cut, name)), name
    assert torch.equal(whole.k_tail[:, :, :300 % 64], cut.k_tail[:, :, :300 % 64])
    assert torch.equal(whole.v_tail[..., :300 % 64], cut.v_tail[..., :300 % 64])


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_at_ties_extremes_and_tiny_values(dtype):
    """Exact halves round to even; a block of zeros is zero; the smallest magnitudes a type has survive."""
    n, smallest = 64 * 4, torch.finfo(dtype).smallest_normal
    k = torch.zeros(1, n, 1, 64, dtype=dtype)
    k[0, :64] = ((torch.arange(64 * 64).reshape(64, 1, 64) % 255 - 127) / 2).to(dtype)
    k[0, 0, 0, 0] = 127.0                                        # scale exactly 1: every half is a tie
    k[0, 64:128] = randn(64, 1, 64, seed=4).to(dtype) * (smallest * 16)
    k[0, 192:256] = randn(64, 1, 64, seed=5).to(dtype) * 200
    v = k.flip(1).contiguous()
    cache = BlockCache(1, 1, 64, n, dtype=dtype)
    cache.append(k.cuda(), v.cuda())
    for codes, scale, x in ((cache.k_codes[0, 0], cache.scales[0, 0, :, 0], k), (cache.v_codes[0, 0].mT, cache.scales[0, 0, :, 1], v)):
        x, s = x[0, :, 0].reshape(4, 64, 64).double(), scale.double().cpu()
        want = (x.abs().amax((1, 2)) / 127).float().double()
        assert torch.equal(s, want)
        code = codes.cpu().double() - 128
        quotient = torch.where(s[:, None, None] > 0, (x.float() / s[:, None, None].float()).double(), 0.0)   # fp32, as defined
        assert torch.equal(code, quotient.round().clamp(-127, 127))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("place", [3, 70, 128])
def test_tokens_that_are_not_finite_touch_only_those_who_see_them(dtype, place):
    k, v = (randn(1, 131, 2, 64, seed=s, dtype=dtype) for s in (1, 2))
    k[0, place, 0, 5] = math.inf
    v[0, place + 1, 1, 63] = math.nan
    cache = BlockCache(1, 2, 64, 200, dtype=dtype)
    cache.append(k.cuda(), v.cuda())
    hk, hv = ref.held(k, v, [131])
    got_k, got_v = cache.read(0, 131)
    assert torch.equal(torch.isnan(got_k).cpu(), torch.isnan(hk)) and not torch.isnan(got_v).any()
    q = randn(1, 131, 4, 64, seed=3, dtype=dtype)
    check_attention(cache, hk, hv, q, causal=True, weights=False)
    check_attention(cache, hk, hv, q[:, -3:], causal=True, weights=False)


def test_rewind_and_append_again():
    k, v = (randn(2, 200, 2, 64, seed=s, dtype=torch.bfloat16).cuda() for s in (1, 2))
    cache = BlockCache(2, 2, 64, 256)
    cache.append(k[:, :100], v[:, :100])
    before = cache.read(0, 100)
    cache.append(k[:, 100:110], v[:, 100:110])
    cache.rewind([100, 104])
    cache.append(k[:, 150:190], v[:, 150:190], counts=[5, 0])
    assert cache.lengths == [105, 104]
    again = cache.read(0, 105)
    assert torch.equal(again[0][:, :100], before[0]) and torch.equal(again[1][:, :100], before[1])
    assert torch.equal(again[0][0, 100:105], k[0, 150:155]) and torch.equal(again[1][1, 100:104], v[1, 100:104])
    assert not again[0][1, 104].any()
    cache.rewind([104, 104])
    cache.append(k[:, 104:128], v[:, 104:128])   # completes the block
    cache.rewind([104, 104])                     # its rows are still there
    cache.append(k[:, 104:200], v[:, 104:200])
    with pytest.raises(ValueError, match="cannot be cut"):
        cache.rewind([110, 200])
    cache.rewind([64, 0])
    assert cache.lengths == [64, 0]


def test_rows_of_tokens_that_were_given_up_are_not_cut_back_to():
    k, v = (randn(1, 256, 1, 64, seed=s, dtype=torch.bfloat16).cuda() for s in (1, 2))
    cache = BlockCache(1, 1, 64, 256)
    cache.append(k[:, :104], v[:, :104])
    cache.rewind([0])
    cache.append(k[:, 128:256], v[:, 128:256])       # block 1 again, complete at once: 16-bit rows of it are the old ones
    with pytest.raises(ValueError, match="cannot be cut"):
        cache.rewind([100])
    cache.rewind([64])
    cache.append(k[:, :20], v[:, :20])
    cache.rewind([70])
    assert torch.equal(cache.read(64, 70)[0], k[:, :6])


def test_rewind_gives_up_the_weights_of_dropped_blocks():
    cache, hk, hv = filled([200], 1, 64, torch.bfloat16, 3)
    cache.weights.fill_(1.0)
    cache.rewind([128])
    assert cache.weights[0, 0, :2].tolist() == [1.0, 1.0] and not cache.weights[0, 0, 2:].any()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rotary_dim", [32, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_keys_rotated_on_the_way_in_are_those_rotated_before(layout, rotary_dim, dtype):
    k, v = (randn(2, 150, 3, 128, seed=s, dtype=dtype).cuda() for s in (1, 2))
    rotary = Rotary(128, 400, rotary_dim=rotary_dim, layout=layout)
    positions = torch.randint(0, 400, (2, 150), generator=torch.Generator().manual_seed(3)).to(torch.int32).cuda()
    inside, before = BlockCache(2, 3, 128, 256, dtype=dtype), BlockCache(2, 3, 128, 256, dtype=dtype)
    inside.append(k, v, rotary=rotary, positions=positions)
    before.append(rotary.apply(k, positions=positions), v)
    for a, b in zip(inside.read(0, 150), before.read(0, 150)):
        assert torch.equal(a, b)


def test_rows_of_any_strides_and_alignment():
    base = randn(2, 90, 8, 130, seed=1, dtype=torch.bfloat16).cuda()
    k, v = base[:, :, 1:7:2, 1:129], base[:, :, 0:6:2, 2:130]          # odd starts, gaps between heads
    rotary = Rotary(128, 90, layout="half")
    positions = torch.arange(90, dtype=torch.int32, device="cuda").expand(2, 90).contiguous()
    odd, plain = BlockCache(2, 3, 128, 128), BlockCache(2, 3, 128, 128)
    odd.append(k, v, rotary=rotary, positions=positions)
    plain.append(k.contiguous(), v.contiguous(), rotary=rotary, positions=positions)
    for a, b in zip(odd.read(0, 90), plain.read(0, 90)):
        assert torch.equal(a, b)
    q = base[:, :40, 1:7, 1:129]
    for a, b in zip(odd.attend(q), plain.attend(q.contiguous())):
        assert torch.equal(a, b)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)                # heads outermost
    for a, b in zip(odd.attend(qt), plain.attend(q.contiguous())):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,group", [(64, 2, 1), (128, 2, 4), (128, 1, 7), (64, 1, 16), (128, 1, 40)])
@pytest.mark.parametrize("lengths", [[1, 2], [63, 64, 65], [128, 300], [777]])
def test_one_query_token(lengths, dim, heads, group, dtype):
    cache, hk, hv = filled(lengths, heads, dim, dtype, 21)
    q = randn(len(lengths), 1, heads * group, dim, seed=7, dtype=dtype, std=1.5)
    check_attention(cache, hk, hv, q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,group,tokens", [(64, 2, 1, 5), (128, 2, 3, 4), (128, 1, 1, 17), (64, 2, 2, 63),
                                                    (128, 1, 2, 130), (128, 2, 1, 257), (64, 1, 4, 300)])
@pytest.mark.parametrize("causal", [True, False])
def test_several_query_tokens(dim, heads, group, tokens, causal, dtype):
    lengths = [tokens, tokens + 3, tokens + 190]
    cache, hk, hv = filled(lengths, heads, dim, dtype, 31)
    q = randn(3, tokens, heads * group, dim, seed=8, dtype=dtype, std=1.5)
    check_attention(cache, hk, hv, q, causal=causal)


@pytest.mark.parametrize("tokens", [3, 40, 150])
@pytest.mark.parametrize("causal", [True, False])
def test_queries_that_see_nothing(tokens, causal):
    """Empty sequences, sequences shorter than the queries, and fewer queries than rows."""
    lengths = [0, 1, 2, 100, 160]
    cache, hk, hv = filled(lengths, 2, 128, torch.bfloat16, 41)
    q = randn(5, tokens, 4, 128, seed=9, dtype=torch.bfloat16)
    check_attention(cache, hk, hv, q, causal=causal)
    check_attention(cache, hk, hv, q, causal=causal, counts=[tokens, 0, 1, tokens - 1, tokens])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 70])
def test_scores_that_rise_by_thousands(tokens, dtype):
    """Every block's scores lie far above those before: the running reference moves at each of them."""
    n = 400
    k, v = randn(1, n, 1, 64, seed=1, dtype=dtype), randn(1, n, 1, 64, seed=2, dtype=dtype)
    k[0, :, 0, 0] = (torch.arange(n) * 2.0).to(dtype)
    q = randn(1, tokens, 2, 64, seed=3, dtype=dtype)
    q[..., 0] = 10.0
    q[:, :, 1, 0] = -10.0                                     # and falls for the other head
    cache = BlockCache(1, 1, 64, n, dtype=dtype)
    cache.append(k.cuda(), v.cuda())
    hk, hv = ref.held(k, v, [n])
    check_attention(cache, hk, hv, q, causal=False, scale=1.0)


@pytest.mark.parametrize("tokens", [1, 5, 140])
def test_blocks_of_very_unlike_scales(tokens):
    """Values from 1e-6 to 1e4 between blocks; the large ones carry little weight."""
    n, dtype = 64 * 6 + 9, torch.bfloat16
    k, v = randn(1, n, 2, 128, seed=1, dtype=dtype), randn(1, n, 2, 128, seed=2, dtype=dtype)
    for i, size in enumerate([1e-6, 1e4, 1.0, 0.0, 1e-3, 50.0, 1e-5]):
        v[0, 64 * i:64 * (i + 1)] *= size
    cache = BlockCache(1, 2, 128, n, dtype=dtype)
    cache.append(k.cuda(), v.cuda())
    check_attention(cache, *ref.held(k, v, [n]), randn(1, tokens, 4, 128, seed=5, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,group", [(1, 1), (1, 5), (2, 8), (60, 1)])
def test_long_sequences_are_split_and_joined(tokens, group, dtype):
    cache, hk, hv = filled([9001, 2500], 2, 128, dtype, 51)
    q = randn(2, tokens, 2 * group, 128, seed=6, dtype=dtype, std=2.0)
    check_attention(cache, hk, hv, q)


def test_results_do_not_change_from_call_to_call():
    cache, _, _ = filled([3000, 1700], 4, 128, torch.bfloat16, 61)
    for tokens in (1, 4, 200):
        q = randn(2, tokens, 16, 128, seed=6, dtype=torch.bfloat16).cuda()
        weights = [torch.zeros_like(cache.weights) for _ in range(3)]
        results = [(*cache.attend(q, weights=w), w) for w in weights]
        for other in results[1:]:
            for a, b in zip(results[0], other):
                assert torch.equal(a, b)


def test_the_tensor_core_kernels_agree_with_the_plain_one():
    cache, _, _ = filled([700, 333], 2, 128, torch.bfloat16, 71)
    for tokens in (1, 200):
        q = randn(2, tokens, 6, 128, seed=6, dtype=torch.bfloat16).cuda()
        out, lse = cache.attend(q)
        ops.force_simt(True)
        try:
            plain, plain_lse = cache.attend(q)
        finally:
            ops.force_simt(False)
        assert float((out.float() - plain.float()).abs().max()) <= 4 * 2.0 ** -8 * float(plain.float().abs().max())
        seen = plain_lse > -math.inf
        assert torch.equal(seen, lse > -math.inf) and float((lse - plain_lse)[seen].abs().max()) < 1e-4


def test_another_stream_and_many_sequences():
    """150 sequences take more than one launch; work goes to the current stream."""
    lengths = [(37 * i) % 140 for i in range(150)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cache, hk, hv = filled(lengths, 1, 64, torch.float16, 81)
        check_attention(cache, hk, hv, randn(150, 1, 2, 64, seed=2, dtype=torch.float16))
        cache.weights.copy_(randn(150, 1, cache.blocks, seed=3).abs())
        cache.evict(1, sinks=0, recent=0)
        side.synchronize()
    assert cache.lengths == [min(n // 64, 1) * 64 + n % 64 for n in lengths]


def test_offsets_past_two_to_the_31():
    """Slots at the far end of arrays of more than 2^31 elements."""
    heads, blocks, dim = 2, 140000, 128
    cache = BlockCache(1, heads, dim, blocks * BLOCK)
    assert cache.k_codes.numel() > 2 ** 31
    cache.table[0, 1, :4] = torch.tensor([blocks - 1, blocks - 2, blocks - 3, blocks - 4], dtype=torch.int32, device="cuda")
    k, v = (randn(1, 200, heads, dim, seed=s, dtype=torch.bfloat16) for s in (1, 2))
    cache.append(k.cuda(), v.cuda())
    hk, hv = ref.held(k, v, [200])
    got = cache.read(0, 200)
    assert ((got[0].double().cpu() - hk).abs() <= 2.0 ** -8 * hk.abs()).all()
    check_attention(cache, hk, hv, randn(1, 1, 4, dim, seed=3, dtype=torch.bfloat16), weights=False)
    check_attention(cache, hk, hv, randn(1, 130, 2, dim, seed=3, dtype=torch.bfloat16), weights=False)


# ------------------------------------------------------------------ eviction
def evicted(weights, table, full, partial, keep, sinks, recent):
    always = [i for i in range(full) if i < sinks or i >= full - recent]
    rest = sorted((i for i in range(full) if i not in always),
                  key=lambda i: (-(math.inf if math.isnan(weights[i]) else weights[i]), not math.isnan(weights[i]), i))
    kept = sorted(always + rest[:max(0, min(keep, full) - len(always))]) + [full] * partial
    freed = [i for i in range(full + partial) if i not in kept]
    order = kept + freed + list(range(full + partial, len(table)))
    return [table[i] for i in order], [weights[i] for i in kept] + [0.0] * (len(table) - len(kept))


@pytest.mark.parametrize("blocks,keep,sinks,recent", [(1, 1, 0, 0), (5, 0, 0, 0), (9, 4, 1, 1), (300, 17, 0, 0), (300, 257, 3, 40),
                                                      (300, 43, 3, 40), (2100, 1000, 1, 8)])
@pytest.mark.parametrize("kind", ["ties", "spread", "odd"])
def test_eviction_keeps_the_heaviest_and_the_lowest_of_equals(blocks, keep, sinks, recent, kind):
    weights = randn(3, 2, blocks, seed=blocks).abs()
    if kind == "ties":
        weights = (weights * 3).round()
    elif kind == "odd":
        weights = randn(3, 2, blocks, seed=blocks)                 # negative ones too
        weights.view(-1)[::7] = math.inf
        weights.view(-1)[3::11] = -0.0
        weights.view(-1)[4::11] = 0.0
        weights.view(-1)[5::13] = math.nan
        weights.view(-1)[6::13] = -math.inf
    table = torch.rand(3, 2, blocks, generator=torch.Generator().manual_seed(1)).argsort(-1).to(torch.int32)
    full, partial = [blocks, blocks - 1, blocks // 2], [0, 1, 1 if blocks > 1 else 0]
    got_table, got_weights = ops.block_evict(weights.cuda(), table.cuda(), full, partial, keep=keep, sinks=sinks, recent=recent)
    for b in range(3):
        for h in range(2):
            want_table, want_weights = evicted(weights[b, h].tolist(), table[b, h].tolist(), full[b], partial[b], keep, sinks, recent)
            assert got_table[b, h].tolist() == want_table
            assert torch.equal(torch.nan_to_num(got_weights[b, h].cpu(), nan=-7.0), torch.nan_to_num(torch.tensor(want_weights), nan=-7.0))


def test_attention_after_eviction_sees_what_was_kept():
    cache, hk, hv = filled([64 * 9 + 20, 64 * 4], 2, 128, torch.bfloat16, 91)
    cache.weights.copy_(randn(2, 2, cache.blocks, seed=4).abs())
    weights = cache.weights.tolist()
    cache.evict(5, sinks=1, recent=1)
    assert cache.lengths == [64 * 5 + 20, 64 * 4]
    new_k, new_v = torch.zeros(2, 64 * 5 + 20, 2, 128, dtype=torch.float64), torch.zeros(2, 64 * 5 + 20, 2, 128, dtype=torch.float64)
    for b, (full, partial) in enumerate([(9, 1), (4, 0)]):
        for h in range(2):
            order, _ = evicted(weights[b][h], list(range(len(weights[b][h]))), full, partial, 5, 1, 1)
            rows = [64 * i + t for i in order[:min(full, 5) + partial] for t in range(64)][:cache.lengths[b]]
            new_k[b, :len(rows), h], new_v[b, :len(rows), h] = hk[b, rows, h], hv[b, rows, h]
    check_attention(cache, new_k, new_v, randn(2, 2, 4, 128, seed=6, dtype=torch.bfloat16), weights=False)
    # and goes on growing: the freed slots are taken again
    k, v = (randn(2, 100, 2, 128, seed=s, dtype=torch.bfloat16) for s in (5, 6))
    cache.append(k.cuda(), v.cuda())
    assert cache.table.sort(-1)[0].eq(torch.arange(cache.blocks, dtype=torch.int32, device="cuda")).all()
    got, _ = cache.read(0, 64 * 5)
    assert ((got[0].double().cpu() - new_k[0, :64 * 5]).abs() <= 2.0 ** -8 * new_k[0, :64 * 5].abs()).all()
