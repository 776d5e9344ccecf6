"""Operators of an 8-bit block cache, as a program that serves with this package calls them.

Every case names a ``path`` and its sizes:

  rotate   queries and keys rotated by their positions (``rotary.Rotary.apply``): half or interleaved pairs, all of a
           head or its first elements, tables scaled for long contexts, and the transposed direction of the gradient.
  store    tokens appended to the cache (``block_cache.BlockCache.append``, keys rotated on the way in where the case
           says so) and the rows of the blocks they touch read back (``BlockCache.read``).
  attend   grouped-head attention over the cache (``BlockCache.attend``), causal or not, with or without the
           accumulation of attention weight per block.
  evict    the blocks of least accumulated weight leave the block table (``ops.block_evict``).

The cache of a sequence and key/value head holds blocks of 64 tokens: 8-bit codes (code + 128) of K as [64, D] and of
V as [D, 64], one fp32 scale each, found through a table of slots; the tokens of the open block are kept in 16 bits,
K as [64, D] and V as [D, 64].
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the positions of one decoding step: 32 sequences, 40 query and 8 key heads, a table scaled for long contexts
        dict(name="rotate_step", path="rotate", batch=32, tokens=1, heads=40, kv_heads=8, dim=128, rotary=128, rows=32768,
             layout="half", scaled=True, transposed=False, dtype="bf16"),
        # the gradient of a long chunk's queries and keys: interleaved pairs in the first half of each head
        dict(name="rotate_chunk_back", path="rotate", batch=1, tokens=24960, heads=24, kv_heads=24, dim=128, rotary=64,
             rows=24960, layout="interleaved", scaled=False, transposed=True, dtype="f16"),
        # one decoding step written: 32 sequences at odd places of their open blocks
        dict(name="store_step", path="store", batch=32, tokens=1, start=8229, kv_heads=8, dim=128, rotate=True, dtype="bf16"),
        # the prefill of a long history, rotated on the way in, with an open block at its end
        dict(name="store_chunk", path="store", batch=1, tokens=24967, start=0, kv_heads=40, dim=128, rotate=True, dtype="bf16"),
        # the smallest read: one query token over a frame and a bit
        dict(name="attend_short", path="attend", batch=1, tokens=1, length=1597, ragged=False, heads=12, kv_heads=12, dim=128,
             causal=True, weights=False, dtype="bf16"),
        # one query token over a layer's whole history, every head with keys of its own
        dict(name="attend_long_step", path="attend", batch=1, tokens=1, length=99840, ragged=False, heads=40, kv_heads=40,
             dim=128, causal=True, weights=False, dtype="bf16"),
        # a decoding step of a batch of unlike lengths, five query heads to a key head, weights accumulated for eviction
        dict(name="attend_batch_step", path="attend", batch=32, tokens=1, length=16411, ragged=True, heads=40, kv_heads=8,
             dim=128, causal=True, weights=True, dtype="bf16"),
        # a few tokens checked at once: five per sequence, four query heads to a key head, narrow heads
        dict(name="attend_few", path="attend", batch=8, tokens=5, length=8191, ragged=True, heads=32, kv_heads=8, dim=64,
             causal=True, weights=False, dtype="f16"),
        # a three-frame chunk of queries over sixteen frames, all of them visible
        dict(name="attend_chunk", path="attend", batch=1, tokens=4680, length=24960, ragged=False, heads=24, kv_heads=24,
             dim=128, causal=False, weights=False, dtype="bf16"),
        # a prompt attended as it was appended: causal, grouped heads, weights accumulated, an open block
        dict(name="attend_prompt", path="attend", batch=2, tokens=4095, length=4095, ragged=False, heads=32, kv_heads=8,
             dim=128, causal=True, weights=True, dtype="f16"),
        # room made in one short sequence's cache
        dict(name="evict_short", path="evict", batch=1, kv_heads=8, blocks=129, keep=96, sinks=1, recent=8),
        # room made in a batch of long caches
        dict(name="evict_batch", path="evict", batch=32, kv_heads=40, blocks=1561, keep=1024, sinks=1, recent=32),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    path = rng.choice(["rotate", "store", "attend", "attend", "attend", "evict"])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 24, 40])
    group = rng.choice([1, 1, 2, 4, 5, 8])
    dim = rng.choice([64, 128, 128])
    if path == "evict":
        blocks = _between(rng, 3, 1600)
        keep = rng.randint(1, blocks)
        sinks = rng.randint(0, min(2, keep))
        return dict(path=path, batch=_between(rng, 1, 32), kv_heads=kv_heads, blocks=blocks, keep=keep, sinks=sinks,
                    recent=rng.randint(0, min(32, keep - sinks)))
    if path == "rotate":
        tokens = _between(rng, 1, 24960)
        batch = _between(rng, 1, max(1, min(32, 24960 // tokens)))
        heads = kv_heads * group if kv_heads * group * tokens * batch <= 24 * 24960 else kv_heads
        heads = heads if heads * tokens * batch <= 24 * 24960 else 1
        return dict(path=path, batch=batch, tokens=tokens, heads=heads, kv_heads=min(heads, kv_heads), dim=dim,
                    rotary=rng.choice([dim, dim, dim // 2, dim // 4]), rows=max(tokens, rng.choice([4096, 32768])),
                    layout=rng.choice(["half", "interleaved"]), scaled=rng.random() < 0.5, transposed=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "f16", "f32"]))
    dtype = rng.choice(["bf16", "f16"])
    if path == "store":
        tokens = 1 if rng.random() < 0.3 else _between(rng, 2, 24960)
        batch = _between(rng, 1, max(1, min(32, 24960 // tokens)))
        # one step may land anywhere in the open block; a chunk starts a block
        start = _between(rng, 1, 9000)
        start = start if tokens == 1 else start // BLOCK * BLOCK
        while kv_heads * batch * tokens > 40 * 24960:
            kv_heads //= 2
        return dict(path=path, batch=batch, tokens=tokens, start=start, kv_heads=max(1, kv_heads), dim=dim,
                    rotate=rng.random() < 0.5, dtype=dtype)
    kind = rng.choice(["step", "step", "few", "chunk"])
    tokens = {"step": 1, "few": rng.randint(2, 16), "chunk": _between(rng, 17, 4680)}[kind]
    length = max(tokens, _between(rng, 1, 99840 if kind == "step" else 24960))
    batch = _between(rng, 1, 32)
    while batch > 1 and batch * length * kv_heads > 40 * 99840:
        batch = batch // 2
    while kv_heads > 1 and batch * length * kv_heads > 40 * 99840:
        kv_heads //= 2
    while batch > 1 and batch * tokens * length * kv_heads * group > 24 * 4680 * 24960:
        batch = batch // 2
    while group > 1 and batch * tokens * length * kv_heads * group > 24 * 4680 * 24960:
        group //= 2
    while kv_heads > 1 and batch * tokens * length * kv_heads * group > 24 * 4680 * 24960:
        kv_heads //= 2
    return dict(path=path, batch=batch, tokens=tokens, length=length, ragged=batch > 1 and rng.random() < 0.6,
                heads=kv_heads * group, kv_heads=kv_heads, dim=dim, causal=rng.random() < 0.7, weights=rng.random() < 0.5,
                dtype=dtype)


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Tokens of every sequence: all alike, or spread evenly between about an eighth of the longest and the longest."""
    n, batch = case["length"], case["batch"]
    if not case["ragged"]:
        return [n] * batch
    return [max(1, n - (n * 7 // 8) * i // max(1, batch - 1) - (i % 3)) if i else n for i in range(batch)]


def _table(rows, rotary, scaled, device):
    """cos and sin of position times frequency, fp32 [rows, rotary/2, 2].  Scaled: frequencies whose wave is longer than
    the 4,096 positions trained on are slowed down eightfold, those with 32 waves and more in them are left, and those
    between are blended; the entries carry the matching temperature."""
    i = torch.arange(rotary // 2, dtype=torch.float64)
    freq = 10000.0 ** (-2.0 * i / rotary)
    gain = 1.0
    if scaled:
        waves = 4096 * freq / (2 * math.pi)
        kept = ((waves - 1) / (32 - 1)).clamp(0, 1)
        freq = freq / 8 * (1 - kept) + freq * kept
        gain = 0.1 * math.log(8) + 1
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return (torch.stack([angle.cos(), angle.sin()], -1) * gain).to(torch.float32).to(device)


def _quantise(x):
    """Codes (plus 128) and scales of blocks whose last two dimensions share a scale."""
    scale = x.float().abs().amax((-2, -1)) / 127
    code = torch.round(x.float() / scale[..., None, None]).clamp(-127, 127)
    return (code + 128).to(torch.uint8), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"

    def normal(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    b = case["batch"]
    if case["path"] == "evict":
        # weights as attention leaves them: long-tailed, with ties at zero among blocks that nobody looked at
        h, p = case["kv_heads"], case["blocks"] + 3
        mass = torch.exp(3 * normal(b, h, p))
        mass = torch.where(torch.rand(b, h, p, generator=gen, device=dev) < 0.2, 0.0, mass)
        table = torch.rand(b, h, p, generator=gen, device=dev).argsort(-1).to(torch.int32)
        return dict(case=case, mass=mass, table=table, full=[max(1, case["blocks"] - i % 3) for i in range(b)],
                    partial=[i % 2 for i in range(b)])
    d, t, dtype = case["dim"], case["tokens"], TYPES[case["dtype"]]
    if case["path"] == "rotate":
        table = _table(case["rows"], case["rotary"], case["scaled"], dev)
        positions = torch.randint(0, case["rows"] - t + 1, (b, 1), generator=gen, device=dev) + torch.arange(t, device=dev)
        state = dict(case=case, table=table, positions=positions.to(torch.int32), q=normal(b, t, case["heads"], d, dtype=dtype),
                     k=normal(b, t, case["kv_heads"], d, dtype=dtype))
        if own:
            from nanokv_b200.rotary import Rotary
            state["rotary"] = Rotary.over(table, head_dim=d, layout=case["layout"])
        return state
    h = case["kv_heads"]
    if case["path"] == "store":
        lengths, p = [case["start"]] * b, (case["start"] + t + BLOCK - 1) // BLOCK + 1
    else:
        lengths = _lengths(case)
        p = (max(lengths) + BLOCK - 1) // BLOCK + 1
    # keys whose channels differ in size, as attention layers have them
    size = torch.exp(0.5 * normal(1, h, 1, 1, d))
    kinds, codes, scales, tails = ("k", "v"), {}, {}, {}
    for kind in kinds:
        x = normal(b, h, p, BLOCK, d) * (size if kind == "k" else 1.0)
        x = x.to(dtype)
        x = x.transpose(-1, -2).contiguous() if kind == "v" else x
        codes[kind], scales[kind] = _quantise(x)
        tails[kind] = x[:, :, 0].contiguous()
    state = dict(case=case, lengths=lengths, k_codes=codes["k"], v_codes=codes["v"],
                 scales=torch.stack([scales["k"], scales["v"]], -1).contiguous(),
                 table=torch.rand(b, h, p, generator=gen, device=dev).argsort(-1).to(torch.int32),
                 k_tail=tails["k"], v_tail=tails["v"])
    if case["path"] == "store":
        state["k"] = normal(b, t, h, d, dtype=dtype)
        state["v"] = normal(b, t, h, d, dtype=dtype)
        state["positions"] = (case["start"] + torch.arange(t, device=dev)).to(torch.int32).expand(b, t).contiguous()
        state["rope"] = _table(case["start"] + t, d, False, dev)
    else:
        state["q"] = normal(b, t, case["heads"], d, dtype=dtype, std=1.5)
    if own:
        from nanokv_b200.block_cache import BlockCache
        from nanokv_b200.rotary import Rotary
        state["cache"] = BlockCache.over(state["k_codes"], state["v_codes"], state["scales"], state["table"],
                                         state["k_tail"], state["v_tail"], lengths)
        if case["path"] == "store":
            state["rotary"] = Rotary.over(state["rope"], head_dim=d, layout="half")
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return {"rotate": _rotate, "store": _store, "attend": _attend, "evict": _evict}[case["path"]](case, state)


def _rotated(x, table, positions, layout, transposed):
    rd = 2 * table.shape[1]
    entry = table[positions.long()][:, :, None]
    c, s = entry[..., 0], -entry[..., 1] if transposed else entry[..., 1]
    xf = x.float()
    turned = xf[..., :rd]
    if layout == "half":
        a, b = turned[..., :rd // 2], turned[..., rd // 2:]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([turned, xf[..., rd:]], -1).to(x.dtype)


def _rotate(case, state):
    if own:
        return state["rotary"].apply(state["q"], state["k"], positions=state["positions"], transposed=case["transposed"])
    return tuple(_rotated(state[n], state["table"], state["positions"], case["layout"], case["transposed"]) for n in "qk")


def _values(codes, scales, slots):
    """Values that the codes of the listed slots stand for: [b, h, blocks, ., .] in 32 bits."""
    index = slots.long()[..., None, None].expand(-1, -1, -1, *codes.shape[3:])
    return (codes.gather(2, index).float() - 128) * scales.gather(2, slots.long())[..., None, None]


def _store(case, state):
    t, start = case["tokens"], case["start"]
    first, stop = start // BLOCK * BLOCK, start + t
    if own:
        cache = state["cache"]
        cache.rewind([start] * case["batch"])
        cache.append(state["k"], state["v"], rotary=state["rotary"] if case["rotate"] else None,
                     positions=state["positions"] if case["rotate"] else None)
        return cache.read(first, stop)
    k, v = state["k"], state["v"]
    if case["rotate"]:
        k = _rotated(k, state["rope"], state["positions"], "half", False)
    held = start - first
    rows = []
    for x, tail in ((k, state["k_tail"]), (v, state["v_tail"].transpose(-1, -2))):
        x = torch.cat([tail[:, :, :held], x.transpose(1, 2)], 2)
        whole = x.shape[2] // BLOCK * BLOCK
        blocks = x[:, :, :whole].unflatten(2, (-1, BLOCK))
        codes, scales = _quantise(blocks)
        kept = ((codes.float() - 128) * scales[..., None, None]).flatten(2, 3).to(x.dtype)
        rows.append(torch.cat([kept, x[:, :, whole:]], 2).transpose(1, 2).contiguous())
    return tuple(rows)


def _attend(case, state):
    q = state["q"]
    if own:
        weights = torch.zeros(state["table"].shape, device=q.device) if case["weights"] else None
        out, lse = state["cache"].attend(q, causal=case["causal"], weights=weights)
        return (out, lse) if weights is None else (out, lse, weights)
    b, t, heads, d = q.shape
    h, lengths, table = case["kv_heads"], state["lengths"], state["table"]
    p = table.shape[2]
    k = _values(state["k_codes"], state["scales"][..., 0], table)
    v = _values(state["v_codes"], state["scales"][..., 1], table).transpose(-1, -2)
    # the open block stands behind the full ones
    n = torch.tensor(lengths, device=q.device)
    is_open = (torch.arange(p, device=q.device) == (n // BLOCK)[:, None])[:, None, :, None, None]
    k = torch.where(is_open, state["k_tail"].float()[:, :, None], k).flatten(2, 3)
    v = torch.where(is_open, state["v_tail"].float().transpose(-1, -2)[:, :, None], v).flatten(2, 3)
    rows = q.float().reshape(b, t, h, heads // h, d).permute(0, 2, 1, 3, 4).reshape(b, h, -1, d)
    s = rows @ k.transpose(-1, -2) / math.sqrt(d)
    seen = n[:, None] - t + 1 + torch.arange(t, device=q.device) if case["causal"] else n[:, None].expand(b, t)
    hidden = torch.arange(p * BLOCK, device=q.device) >= seen.repeat_interleave(heads // h, 1)[:, None, :, None]
    s.masked_fill_(hidden, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    out = (w @ v) / torch.where(total == 0, 1.0, total)
    lse = (top + total.log()).squeeze(-1)

    def back(x):
        return x.reshape(b, h, t, heads // h, *x.shape[3:]).transpose(1, 2).flatten(2, 3).contiguous()

    if not case["weights"]:
        return back(out).to(q.dtype), back(lse)
    share = w.div_(torch.where(total == 0, 1.0, total)).sum(2).unflatten(-1, (p, BLOCK)).sum(-1)
    return back(out).to(q.dtype), back(lse), share


def _evict(case, state):
    mass, table = state["mass"], state["table"]
    keep, sinks, recent = case["keep"], case["sinks"], case["recent"]
    if own:
        from nanokv_b200 import ops
        return ops.block_evict(mass, table, state["full"], state["partial"], keep=keep, sinks=sinks, recent=recent)
    b, h, p = mass.shape
    at = torch.arange(p, device=mass.device)
    full = torch.tensor(state["full"], device=mass.device)[:, None, None]
    partial = torch.tensor(state["partial"], device=mass.device)[:, None, None]
    forced = (at < sinks) | (at >= full - recent)
    key = torch.where(forced, math.inf, mass)
    key = torch.where(at < full, key, -math.inf)
    rank = key.sort(dim=-1, descending=True, stable=True)[1].argsort(-1)
    kept = ((rank < keep) & (at < full)) | ((at == full) & (partial == 1))
    live = at < full + partial
    # kept ones in order, the freed behind them, the unused last
    order = torch.where(kept, 0, torch.where(live, 1, 2)).sort(dim=-1, stable=True)[1]
    moved = torch.where(kept, mass, 0.0)
    return table.gather(2, order), moved.gather(2, order)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b, size = case["batch"], {"bf16": 2, "f16": 2, "f32": 4}.get(case.get("dtype"), 4)
    if case["path"] == "evict":
        entries = b * case["kv_heads"] * (case["blocks"] + 3)
        return {"bytes": 16 * entries, "flops": entries}
    t, d, h = case["tokens"], case["dim"], case["kv_heads"]
    if case["path"] == "rotate":
        n = b * t * (case["heads"] + h) * d
        return {"bytes": 2 * n * size + b * t * 4 + min(case["rows"], b * t) * case["rotary"] * 4,
                "flops": 3 * n * case["rotary"] // d}
    if case["path"] == "store":
        first, stop = case["start"] // BLOCK * BLOCK, case["start"] + t
        held, whole = case["start"] - first, stop // BLOCK * BLOCK - first
        per = 2 * b * h * d
        fresh = stop - first - whole if whole else t          # new rows of the open block
        # new rows and those already in the open block read; completed blocks' codes written and read with their
        # scales; new open rows written and read; rows handed back; cosines and sines of the positions
        return {"bytes": per * (2 * t + 2 * held + 2 * whole + 4 * fresh + 2 * (stop - first))
                + 2 * 8 * b * h * (whole // BLOCK) + (t * d * 4 if case["rotate"] else 0),
                "flops": per * (t * (3 if case["rotate"] else 0) // 2 + 4 * (stop - first))}
    lengths, heads = _lengths(case), case["heads"]
    seen = sum(sum(max(0, n - t + i + 1) for i in range(t)) if case["causal"] else n * t for n in lengths)
    n = sum(lengths)
    tails = sum(x % BLOCK for x in lengths)
    return {"bytes": 2 * b * t * heads * d * size + 4 * b * t * heads + 2 * n * h * d + 2 * tails * h * d
            + 8 * h * (n // BLOCK) + (8 * h * (n // BLOCK) if case["weights"] else 0),
            "flops": 4 * seen * heads * d}


# ------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["path"] == "evict":
        return _exact_evict(case, state)
    if case["path"] == "rotate":
        return tuple(_exact_rotated(state[n], state["table"], state["positions"], case["layout"], case["transposed"])
                     for n in "qk")
    return _exact_store(case, state) if case["path"] == "store" else _exact_attend(case, state)


def _exact_rotated(x, table, positions, layout, transposed):
    """The rotation as a product of complex numbers."""
    turn = torch.view_as_complex(table.double())[positions.long()][:, :, None]
    turn = turn.conj() if transposed else turn
    y = x.double().clone()
    rd = 2 * table.shape[1]
    if layout == "half":
        z = torch.complex(y[..., :rd // 2], y[..., rd // 2:rd]) * turn
        y[..., :rd // 2], y[..., rd // 2:rd] = z.real, z.imag
    else:
        z = torch.complex(y[..., 0:rd:2], y[..., 1:rd:2]) * turn
        y[..., 0:rd:2], y[..., 1:rd:2] = z.real, z.imag
    return y


def _exact_store(case, state):
    start, t = case["start"], case["tokens"]
    held, dtype = start % BLOCK, state["k"].dtype
    results = []
    for kind in "kv":
        new = state[kind].double()
        if kind == "k" and case["rotate"]:
            # the cache holds rotated keys in its own type
            new = _exact_rotated(state["k"], state["rope"], state["positions"], "half", False).to(dtype).double()
        tail = state["k_tail"] if kind == "k" else state["v_tail"].mT
        rows = torch.cat([tail[:, :, :held].permute(0, 2, 1, 3).double(), new], 1)
        for at in range(0, rows.shape[1] - BLOCK + 1, BLOCK):
            block = rows[:, at:at + BLOCK]
            step = block.abs().amax((1, 3), keepdim=True) / 127
            block.copy_((block / step).round() * step)
        results.append(rows)
    return tuple(results)


def _exact_attend(case, state):
    q, table, lengths = state["q"].double(), state["table"].long(), state["lengths"]
    b, t, heads, d = q.shape
    h, group = case["kv_heads"], heads // case["kv_heads"]
    out = torch.zeros_like(q)
    lse = torch.full((b, t, heads), -math.inf, dtype=torch.float64, device=q.device)
    shares = torch.zeros(table.shape, dtype=torch.float64, device=q.device)
    if b * h > 2048:
        return None
    for i in range(b):
        n, full = lengths[i], lengths[i] // BLOCK
        for j in range(h):
            slots = table[i, j, :full]
            step = state["scales"][i, j].double()[slots]
            k = (state["k_codes"][i, j].index_select(0, slots).double() - 128) * step[:, 0, None, None]
            v = (state["v_codes"][i, j].index_select(0, slots).double() - 128) * step[:, 1, None, None]
            k = torch.cat([k.reshape(-1, d), state["k_tail"][i, j, :n - full * BLOCK].double()])
            v = torch.cat([v.mT.reshape(-1, d), state["v_tail"][i, j, :, :n - full * BLOCK].double().mT])
            for g in range(group):
                head = j * group + g
                for a in range(0, t, 1024):
                    s = q[i, a:a + 1024, head] @ k.T * d ** -0.5
                    if case["causal"]:
                        last = torch.arange(a, a + s.shape[0], device=q.device) + n - t
                        s = torch.where(torch.arange(n, device=q.device) <= last[:, None], s, -math.inf)
                    total = torch.logsumexp(s, -1)
                    w = torch.nan_to_num(torch.exp(s - total[:, None]), nan=0.0)
                    out[i, a:a + 1024, head] = w @ v
                    lse[i, a:a + 1024, head] = total
                    sums = torch.nn.functional.pad(w.sum(0), (0, table.shape[2] * BLOCK - n))
                    shares[i, j] += sums.reshape(-1, BLOCK).sum(-1)
    return (out, lse, shares) if case["weights"] else (out, lse)


def _exact_evict(case, state):
    tables, weights = state["table"].tolist(), state["mass"].double().tolist()
    for i, (n, partial) in enumerate(zip(state["full"], state["partial"])):
        for table, mass in zip(tables[i], weights[i]):
            always = {x for x in range(n) if x < case["sinks"] or x >= n - case["recent"]}
            others = sorted((x for x in range(n) if x not in always), key=lambda x: (-mass[x], x))
            kept = sorted(always | set(others[:max(0, case["keep"] - len(always))])) + [n] * partial
            freed = sorted(set(range(n + partial)) - set(kept))
            order = kept + freed + list(range(n + partial, len(table)))
            table[:] = [table[x] for x in order]
            mass[:] = [mass[x] for x in kept] + [0.0] * (len(mass) - len(kept))
    return (torch.tensor(tables, dtype=torch.int32), torch.tensor(weights, dtype=torch.float64))
