"""The paged 16-bit cache with drafted tokens from its formulas, in 64 bits and token by token."""
import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # relative rounding error


def randn(*shape, seed, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def scattered(batch, capacity, page, seed, spare=3):
    """A table [batch, entries] whose pages are scattered over a pool, and the pool's size."""
    entries = -(-capacity // page)
    pages = batch * entries + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    return order[:batch * entries].reshape(batch, entries).to(torch.int32), pages


def rows_of(pool, table, b, tokens):
    """Tokens [0, tokens) of sequence b: [tokens, kv_heads, D]."""
    page = pool.shape[2]
    t = torch.arange(tokens)
    return pool[table[b].long()[t // page], :, t % page]


def put(pool, table, b, first, rows):
    """rows [n, kv_heads, D] as tokens first, first + 1, ... of sequence b."""
    page = pool.shape[2]
    for i, row in enumerate(rows):
        pool[int(table[b, (first + i) // page]), :, (first + i) % page] = row


def chain(tokens):
    return torch.arange(-1, tokens - 1, dtype=torch.int32)


def tree(tokens, seed):
    """Parents of a random draft: any earlier node, or none."""
    gen = torch.Generator().manual_seed(seed)
    return torch.tensor([int(torch.randint(-1, i, (1,), generator=gen)) if i else -1 for i in range(tokens)], dtype=torch.int32)


def sees(parents):
    """[T, T] bool: the ancestors of every node, and itself."""
    out = torch.zeros(len(parents), len(parents), dtype=torch.bool)
    for i, p in enumerate(parents.tolist()):
        if p >= 0:
            out[i] = out[p]
        out[i, i] = True
    return out


def packed(mask):
    """Bits [.., T, ceil(T / 32)] i32 of a mask [.., T, T]."""
    t = mask.shape[-1]
    bits = torch.nn.functional.pad(mask, (0, -t % 32)).unflatten(-1, (-1, 32)).long()
    words = (bits << torch.arange(32)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def attention(q, k_pages, v_pages, table, lengths, counts, mask, scale):
    """q [B,T,Hq,D]; mask [B,T,T] bool over the pending tokens -> out, lse, spread [B,T,Hq,D] (sum of p |v|) and size
    [B,T,Hq] (largest sum of |q| |k| times |scale|).  What a query does not see has no part in its result."""
    q = q.double().cpu()
    B, T, Hq, D = q.shape
    H = k_pages.shape[1]
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    lse, size = torch.full((B, T, Hq), -math.inf, dtype=torch.float64), torch.zeros(B, T, Hq, dtype=torch.float64)
    for b in range(B):
        n, c = lengths[b], counts[b]
        if c == 0 or n + c == 0:
            continue
        k, v = (rows_of(pool, table, b, n + c).double() for pool in (k_pages, v_pages))
        allowed = torch.ones(c, n + c, dtype=torch.bool)
        allowed[:, n:] = mask[b, :c, :c]
        for h in range(Hq):
            kv = h // (Hq // H)
            s = torch.where(allowed, q[b, :c, h] @ k[:, kv].nan_to_num().T * scale, -math.inf)
            poisoned = allowed & (q[b, :c, h][:, None] * k[None, :, kv]).isnan().any(-1)
            s = torch.where(poisoned, math.nan, s)
            total = torch.logsumexp(s, -1)
            lse[b, :c, h] = total
            p = torch.where(total[:, None] == -math.inf, 0.0, torch.exp(s - total[:, None]))
            p = torch.where(allowed, p, 0.0)
            vv = v[:, kv]
            finite = vv.isfinite()
            held = torch.where(finite, vv, 0.0)
            got = p @ held
            for j in (~finite).any(-1).nonzero().flatten().tolist():
                got = got + torch.where((allowed[:, j] & (p[:, j] > 0))[:, None] & ~finite[j], vv[j], 0.0)
            out[b, :c, h], spread[b, :c, h] = got, p @ held.abs()
            big = q[b, :c, h].abs() @ k[:, kv].nan_to_num(posinf=0, neginf=0).abs().T * abs(scale)
            size[b, :c, h] = torch.where(allowed, big, 0.0).amax(-1)
    return out, lse, spread, size
