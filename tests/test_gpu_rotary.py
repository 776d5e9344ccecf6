"""Rotary positions on the GPU against the formula in 64 bits, and their gradient."""
import math

import pytest
import torch

import block_reference as ref
from nanokv_b200.rotary import Rotary

pytestmark = pytest.mark.gpu


def randn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary_dim,batch,tokens,heads,kv_heads", [
    (128, 128, 1, 1, 1, 1), (128, 64, 3, 5, 6, 2), (64, 32, 2, 33, 4, 1), (80, 24, 2, 3, 3, 1), (13, 6, 1, 7, 2, 2),
    (96, 96, 1, 700, 12, 12), (256, 64, 2, 9, 5, 0), (128, 128, 4, 900, 9, 3)])
@pytest.mark.parametrize("transposed", [False, True])
def test_against_the_formula(dtype, layout, dim, rotary_dim, batch, tokens, heads, kv_heads, transposed):
    rotary = Rotary(dim, 5000, rotary_dim=rotary_dim, layout=layout, scaling=dict(kind="blend", factor=4.0, trained=1024))
    q, k = randn(batch, tokens, heads, dim, seed=1, dtype=dtype), randn(batch, tokens, max(kv_heads, 1), dim, seed=2, dtype=dtype)
    positions = torch.randint(0, 5000, (batch, tokens), generator=torch.Generator().manual_seed(3)).to(torch.int32)
    if kv_heads:
        got = rotary.apply(q.cuda(), k.cuda(), positions=positions.cuda(), transposed=transposed)
    else:
        got = (rotary.apply(q.cuda(), positions=positions.cuda(), transposed=transposed),)
    table = rotary.table.cpu()
    for x, y in zip((q, k), got):
        want = ref.rotated(x, table, positions, layout, transposed)
        # two products and a sum in fp32 (each of magnitudes up to 1.2 max|x|), then one rounding to the type
        bound = ref.UNIT[dtype] * want.abs() + 2.0 ** -22 * 1.2 * float(x.float().abs().max())
        assert ((y.double().cpu() - want).abs() <= bound).all()
        assert torch.equal(y.cpu()[..., rotary_dim:], x[..., rotary_dim:])


def test_positions_outside_the_table_are_nan():
    rotary = Rotary(64, 10, rotary_dim=32)
    x = randn(1, 4, 2, 64, seed=1)
    y = rotary.apply(x.cuda(), positions=torch.tensor([[0, -1, 10, 9]], dtype=torch.int32).cuda()).cpu()
    assert torch.isnan(y[0, 1:3, :, :32]).all() and torch.equal(y[0, 1:3, :, 32:], x[0, 1:3, :, 32:])
    assert not torch.isnan(y[0, ::3]).any()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides(layout):
    base = randn(2, 20, 6, 130, seed=1, dtype=torch.bfloat16).cuda()
    rotary = Rotary(128, 64, layout=layout)
    positions = torch.arange(40, dtype=torch.int32, device="cuda").reshape(2, 20)
    for view in (base[:, :, ::2, 1:129], base[..., :128].transpose(1, 2).contiguous().transpose(1, 2), base[:, :, 1:4, 2:130]):
        assert torch.equal(rotary.apply(view, positions=positions), rotary.apply(view.contiguous(), positions=positions))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_the_transposed_direction_is_the_gradient(layout):
    """sum(g * f(x)) has the gradient that the transposed direction gives g, by the formula and by differences."""
    rotary = Rotary(64, 100, rotary_dim=48, layout=layout, scaling=dict(kind="blend", factor=8.0, trained=50))
    positions = torch.tensor([[3, 77, 99]], dtype=torch.int32).cuda()
    x, g = randn(1, 3, 2, 64, seed=1).cuda(), randn(1, 3, 2, 64, seed=2).cuda()
    back = rotary.apply(g, positions=positions, transposed=True)
    leaf = x.cpu().double().requires_grad_()
    (ref.rotated_for_grad(leaf, rotary.table.cpu(), positions.cpu(), layout) * g.cpu().double()).sum().backward()
    # fp32 products and sums of magnitudes below 8: a few units of 2^-22
    assert float((back.cpu().double() - leaf.grad).abs().max()) <= 2.0 ** -18
    for at in [(0, 0, 0, 0), (0, 1, 1, 25), (0, 2, 0, 47), (0, 2, 1, 60)]:
        up, down = x.clone(), x.clone()
        up[at] += 0.5
        down[at] -= 0.5
        # the function is linear: the difference over a step of one is the derivative up to fp32 rounding of the sums
        slope = ((rotary.apply(up, positions=positions) - rotary.apply(down, positions=positions)).double() * g.double()).sum()
        assert math.isclose(float(slope), float(back[at]), abs_tol=2.0 ** -16)
