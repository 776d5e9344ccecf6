"""Attention over blocks whose value scales lie far apart, or at the ends of what 16-bit numbers reach."""
import math

import pytest
import torch

import block_reference as ref
from nanokv_b200 import ops
from nanokv_b200.block_cache import BlockCache

pytestmark = pytest.mark.gpu


def randn(*shape, seed, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def check(k, v, q, *, causal=True, scale=None, least=0.0, weights=True):
    """One call over a cache of rows k, v against the formula in 64 bits.  Bounds: the result's own rounding; the weights'
    rounding to 16 bits (relative, once for the weight and once for the reference point it stands against) times the sum of
    p |v|; scores as fp32 sums of at most 128 products, a relative 2^-18 of the sum of magnitudes, in the weights' exponents.
    ``least``: what values next to the block's type's smallest numbers may lose, absolutely."""
    B, n, H, D = k.shape
    T = q.shape[1]
    cache = BlockCache(B, H, D, n + 64, dtype=k.dtype)
    cache.append(k.cuda(), v.cuda())
    given = torch.zeros_like(cache.weights)
    out, lse = cache.attend(q.cuda(), causal=causal, scale=scale, weights=given if weights else None)
    ops.check_status(out.device)
    hk, hv = ref.held(k, v, [n] * B)
    want, want_lse, spread, size, shares = ref.attention(q, hk, hv, [n] * B, [T] * B, causal, D ** -0.5 if scale is None else scale)
    out, lse, unit = out.double().cpu(), lse.double().cpu(), ref.UNIT[k.dtype]
    assert torch.isfinite(want).all() and torch.isfinite(want_lse).all()
    score = 2.0 ** -18 * size.clamp_min(1.0)
    bad = (lse - want_lse).abs() / (score + 2.0 ** -22 * want_lse.abs())
    assert torch.isfinite(lse).all() and (bad <= 1).all(), float(bad.max())
    bad = (out - want).abs() / (unit * want.abs() + (2 * unit + 4 * score[..., None]) * spread + least)
    assert torch.isfinite(out).all() and (bad <= 1).all(), float(bad.max())
    if weights:
        got, worst = given.double().cpu()[:, :, :shares.shape[2]], float(score.max())
        assert ((got - shares).abs() <= 4 * worst * shares + 2.0 ** -22).all()


TOKENS = [1, 5, 140]          # few rows, and more than either kernel for few rows takes


def sized(n, sizes, seed, heads=2, dim=128, dtype=torch.bfloat16):
    """Values whose blocks are of these sizes."""
    v = randn(1, n, heads, dim, seed=seed)
    for i, size in enumerate(sizes):
        v[:, 64 * i:64 * (i + 1)] *= size
    return v.to(dtype)


@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1e-37, 1e-38, 1e-39])
def test_a_block_of_tiny_values_among_others(size, dim, tokens):
    """bf16 reaches far below the scales whose reciprocals are fp32 numbers; some of the rows do not see the tiny blocks."""
    n = 64 * 7 + 20
    v = sized(n, [1.0, size, 1.0, 1.0, 1.0, size, 1.0, 1.0], 2, dim=dim)
    k, q = (randn(1, m, h, dim, seed=s, dtype=torch.bfloat16) for m, h, s in ((n, 2, 1), (tokens, 4, 3)))
    check(k, v, q, least=2.0 ** -133)


@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("blocks", [2, 7])
@pytest.mark.parametrize("size", [1e-30, 1e-37, 1e-38])
def test_nothing_but_tiny_values(size, blocks, tokens):
    n = 64 * blocks
    v = sized(n, [size] * blocks, 2)
    k, q = (randn(1, m, h, 128, seed=s, dtype=torch.bfloat16) for m, h, s in ((n, 2, 1), (tokens, 4, 3)))
    # two steps of the smallest bf16 number: the result's own rounding there and the weights'
    check(k, v, q, causal=tokens < n, least=2.0 ** -132)


@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("sizes", [[1e30, 1e-30, 1.0, 1e30], [1e-30, 1e-30, 1e30, 0.0], [0.0, 1e36, 0.0, 1.0], [1e-38, 1e30, 1e-38, 1e-38]])
def test_scales_further_apart_than_fp32_reaches(sizes, tokens):
    """The share of a block in the sum and in the block weights does not depend on the size of its values."""
    n = 64 * 4
    k, q = (randn(1, m, h, 128, seed=s, dtype=torch.bfloat16) for m, h, s in ((n, 2, 1), (tokens, 4, 3)))
    check(k, sized(n, sizes, 2), q, least=2.0 ** -133)


@pytest.mark.parametrize("tokens", TOKENS)
def test_small_values_with_the_largest_scores(tokens):
    """Scores rise by 60 and more from block to block while the values get smaller: the sum follows the scores, the result
    what the values leave."""
    n, dim = 64 * 6, 64
    k, q = randn(1, n, 1, dim, seed=1, std=0.1), randn(1, tokens, 2, dim, seed=3, std=0.1)
    k[..., 0] = torch.arange(n)[None, :, None] // 64 * 10.0
    q[..., 0] = 8.0
    v = sized(n, [10.0 ** (-7 * i) for i in range(6)], 2, heads=1, dim=dim)
    check(k.to(torch.bfloat16), v, q.to(torch.bfloat16), causal=False, scale=1.0, least=2.0 ** -126)


# batch and kv heads: enough of them that one worker of either kernel takes many blocks of one head
@pytest.mark.parametrize("batch,heads,n,tokens,dtype", [(8, 40, 8192, 1, torch.bfloat16), (8, 40, 8192, 1, torch.float16),
                                                        (8, 40, 8192, 3, torch.bfloat16), (8, 40, 8192, 3, torch.float16),
                                                        (1, 1, 30000, 140, torch.bfloat16), (1, 40, 8192, 140, torch.bfloat16),
                                                        (1, 40, 8192, 140, torch.float16)])
@pytest.mark.parametrize("nats", [14.0, 18.0])
def test_many_keys_far_below_one(nats, batch, heads, n, tokens, dtype):
    """One key takes all but a little of every row and has no value; the result is what thousands of others leave."""
    dim = 64
    k, q, v = (randn(batch, n, heads, dim, seed=1, std=0.3), randn(batch, tokens, 2 * heads, dim, seed=3, std=0.3),
               1 + randn(batch, n, heads, dim, seed=2))
    k[..., 0], q[..., 0] = 0.0, 8.0
    k[:, 1000, :, 0], v[:, 1000] = nats / 8, 0.0
    # fp16 holds a weight to 2^-25 at worst, of numbers that reach 2^7 at least where the largest weight is 1
    check(k.to(dtype), v.to(dtype), q.to(dtype), causal=False, scale=1.0, least=n * 2.0 ** -32 * float(v.abs().max()))


@pytest.mark.parametrize("batch,heads,tokens", [(32, 40, 1), (32, 40, 4), (1, 1, 140)])
@pytest.mark.parametrize("large", [1e6, 1e8, 1e12])
def test_large_values_under_small_weights(large, batch, heads, tokens):
    """Keys 18 nats lower whose values are larger by as much and more: the result is theirs as well."""
    n, dim = 64 * 6 + 10, 64
    k, q = randn(batch, n, heads, dim, seed=1, std=0.3), randn(batch, tokens, 2 * heads, dim, seed=3, std=0.3)
    k[..., 0], q[..., 0] = 3.0, 6.0
    k[:, 64:128, :, 0] = k[:, 256:320, :, 0] = 0.0
    v = randn(batch, n, heads, dim, seed=2)
    v[:, 64:128] *= large
    v[:, 256:320] *= large
    check(k.to(torch.bfloat16), v.to(torch.bfloat16), q.to(torch.bfloat16), causal=False, scale=1.0)


@pytest.mark.parametrize("tokens", TOKENS)
def test_unlike_scales_in_fp16(tokens):
    """Blocks whose values are 2^-14 and 2^-20 of others', some of them with the larger weights."""
    n, dim = 64 * 7 + 10, 64
    k, q = randn(1, n, 1, dim, seed=1, std=0.3), randn(1, tokens, 2, dim, seed=3, std=0.3)
    k[..., 0], q[..., 0] = 0.0, 4.0
    k[:, 64:128, :, 0] = 2.0
    v = sized(n, [1.0, 2.0 ** -14, 2.0 ** -20, 100.0, 2.0 ** -14, 0.0, 2.0 ** -10, 1.0], 2, heads=1, dim=dim, dtype=torch.float16)
    check(k.to(torch.float16), v, q.to(torch.float16), causal=tokens == 140, scale=1.0, least=n * 2.0 ** -32 * float(v.abs().max()))


@pytest.mark.parametrize("tokens", [1, 140])
@pytest.mark.parametrize("held", [1, 2, 33, 63])
@pytest.mark.parametrize("size", [1e36, 1e30, 1e-30, 1e-39, 0.0])
def test_an_open_block_of_any_size(size, held, tokens):
    """Values of the open block far above and far below the others'; what lies behind its last token is left over."""
    n, dim = 64 * 3 + held, 128
    v = sized(n, [1.0, 1.0, 1.0, size], 2)
    k, q = (randn(1, m, h, dim, seed=s, dtype=torch.bfloat16) for m, h, s in ((n, 2, 1), (tokens, 4, 3)))
    check(k, v, q, least=2.0 ** -133)
