"""The 8-bit block cache and rotary positions from their formulas, in 64 bits and token by token."""
import math

import torch

BLOCK = 64
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # relative rounding error


def rotated(x, table, positions, layout, transposed=False):
    """x [B,T,H,D] (any type) -> f64; positions outside the table give NaN."""
    y, rd = x.double().clone(), 2 * table.shape[1]
    inside = (positions >= 0) & (positions < table.shape[0])
    entry = table.double()[positions.clamp(0, table.shape[0] - 1).long()]
    entry = torch.where(inside[..., None, None], entry, math.nan)[:, :, None]
    c, s = entry[..., 0], entry[..., 1] * (-1 if transposed else 1)
    first = torch.arange(rd // 2) if layout == "half" else torch.arange(0, rd, 2)
    second = first + (rd // 2 if layout == "half" else 1)
    a, b = x.double()[..., first], x.double()[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    return y


def held(k, v, lengths):
    """What a cache holds of rows k, v [B,N,H,D] (16-bit): values f64 [B,N,H,D] each, rows past a length zero; tokens that
    are not finite NaN in K and zero in V, blocks likewise."""
    k, v = k.double().cpu().clone(), v.double().cpu().clone()
    out_k, out_v = torch.zeros_like(k), torch.zeros_like(v)
    bad = ~(torch.isfinite(k).all(-1) & torch.isfinite(v).all(-1))
    k[bad], v[bad] = math.nan, 0.0
    for b, n in enumerate(lengths):
        for t0 in range(0, n, BLOCK):
            stop = min(n, t0 + BLOCK)
            kb, vb = k[b, t0:stop], v[b, t0:stop]
            if stop - t0 == BLOCK:
                bad_heads = torch.isnan(kb).any(-1).any(0)
                kb, vb = quantised(kb), quantised(vb)
                kb[:, bad_heads], vb[:, bad_heads] = math.nan, 0.0
            out_k[b, t0:stop], out_v[b, t0:stop] = kb, vb
    return out_k, out_v


def quantised(x):
    """One block [64,H,D]: rounded to multiples of each head's largest magnitude / 127.  Scale and quotient are fp32 numbers:
    half the largest magnitude is 63.5 steps, which the rounding of the scale would push to one side in 64 bits."""
    scale = (x.abs().amax((0, 2), keepdim=True) / 127).float()
    code = (x.float() / scale).round().clamp(-127, 127).double()
    return torch.where(scale > 0, code * scale.double(), 0.0)


def attention(q, k, v, lengths, counts, causal, scale):
    """q [B,T,Hq,D], values k, v [B,N,H,D] f64 -> out, lse, spread [B,T,Hq,D] (sum of p |v|), size [B,T,Hq] (largest sum of
    |q||k| times scale) and block weights [B,H,ceil(N/64)]."""
    q = q.double().cpu()
    B, T, Hq, D = q.shape
    N, H = k.shape[1], k.shape[2]
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    lse, size = torch.full((B, T, Hq), -math.inf, dtype=torch.float64), torch.zeros(B, T, Hq, dtype=torch.float64)
    shares = torch.zeros(B, H, -(-max(N, 1) // BLOCK) * BLOCK, dtype=torch.float64)
    for b in range(B):
        for h in range(Hq):
            kv = h // (Hq // H)
            s_all = q[b, :, h] @ k[b, :, kv].T * scale
            m_all = q[b, :, h].abs() @ k[b, :, kv].abs().T * scale
            for i in range(T):
                n = lengths[b] if not causal else max(0, min(lengths[b], lengths[b] - counts[b] + i + 1))
                if i >= counts[b] or n == 0:
                    continue
                s = s_all[i, :n]
                lse[b, i, h] = torch.logsumexp(s, 0)
                p = torch.exp(s - lse[b, i, h])
                out[b, i, h], spread[b, i, h] = p @ v[b, :n, kv], p @ v[b, :n, kv].abs()
                size[b, i, h] = m_all[i, :n].max()
                shares[b, kv, :n] += p
    return out, lse, spread, size, shares.unflatten(-1, (-1, BLOCK)).sum(-1)


def rotated_for_grad(x, table, positions, layout):
    """``rotated`` without writes in place, for differentiation."""
    rd = 2 * table.shape[1]
    entry = table.double()[positions.long()][:, :, None]
    c, s = entry[..., 0], entry[..., 1]
    if layout == "half":
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([turned, x[..., rd:]], -1)
