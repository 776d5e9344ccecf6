"""Operators of a paged 16-bit cache with drafted tokens, as a program that serves with this package calls them.

Every case names a ``path`` and its sizes:

  append   pending tokens written behind what the sequences hold (``page_cache.PageCache.append``): keys and queries rotated by
           their positions on the way, keys and values into the pages that the sequences' table names.
  attend   grouped-head attention of the pending tokens over the cache and one another (``PageCache.attend``): a tree of
           drafted tokens, a chain (causal), or all of them visible.
  keep     the rows of the accepted path moved to the front of the pending tokens, several layers at once
           (``page_cache.keep``).
  tree     which drafted tokens every drafted token sees, as bits, and its depth (``ops.tree_mask``).

Keys and values lie in pages [pages, kv_heads, page, D] of one pool; token j of a sequence is row j % page of the page in
entry j / page of its row of the table.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decoding step of a batch: queries and keys of 32 sequences turned, keys and values stored
        dict(name="append_step", path="append", batch=32, tokens=1, length=1597, ragged=True, heads=40, kv_heads=8, dim=128,
             page=64, rotary=128, layout="half", counts=False, dtype="bf16"),
        # the prefill of a long history in one call, large pages, as many query as key heads
        dict(name="append_chunk", path="append", batch=1, tokens=24967, length=0, ragged=False, heads=40, kv_heads=40, dim=128,
             page=128, rotary=128, layout="half", counts=False, dtype="bf16"),
        # the smallest read: one query token over a frame and a bit, every head with keys of its own
        dict(name="attend_short", path="attend", batch=1, tokens=1, length=1596, ragged=False, heads=12, kv_heads=12, dim=128,
             page=64, mask="causal", counts=False, dtype="bf16"),
        # one query token over a layer's whole history
        dict(name="attend_long_step", path="attend", batch=1, tokens=1, length=99839, ragged=False, heads=40, kv_heads=40,
             dim=128, page=64, mask="causal", counts=False, dtype="bf16"),
        # a batch of small trees, sixteen nodes each, over histories of unlike lengths; five query heads to a key head, small pages
        dict(name="attend_batch_tree", path="attend", batch=32, tokens=16, length=16411, ragged=True, heads=40, kv_heads=8,
             dim=128, page=16, mask="tree", counts=True, dtype="bf16"),
        # a wide tree checked at once: 63 nodes, four query heads to a key head, narrow heads
        dict(name="attend_wide_tree", path="attend", batch=8, tokens=63, length=8191, ragged=True, heads=32, kv_heads=8, dim=64,
             page=32, mask="tree", counts=False, dtype="f16"),
        # a three-frame chunk of queries over thirteen frames and itself, all of it visible
        dict(name="attend_chunk", path="attend", batch=1, tokens=4680, length=20280, ragged=False, heads=24, kv_heads=24,
             dim=128, page=128, mask="all", counts=False, dtype="bf16"),
        # a prompt attended as it was appended: causal, grouped heads
        dict(name="attend_prompt", path="attend", batch=2, tokens=4095, length=0, ragged=False, heads=32, kv_heads=8, dim=128,
             page=64, mask="causal", counts=False, dtype="f16"),
        # the accepted tokens of one sequence and layer
        dict(name="keep_short", path="keep", batch=1, tokens=16, length=1597, ragged=False, kv_heads=8, dim=128, page=64,
             accepted=4, layers=1, dtype="bf16"),
        # the accepted tokens of a batch in all layers of a model
        dict(name="keep_layers", path="keep", batch=32, tokens=63, length=301, ragged=True, kv_heads=8, dim=128, page=64,
             accepted=9, layers=40, dtype="bf16"),
        # one draft of sixteen nodes
        dict(name="tree_one", path="tree", batch=1, tokens=16),
        # a batch of large drafts
        dict(name="tree_batch", path="tree", batch=32, tokens=511),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    path = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "keep", "tree"])
    if path == "tree":
        return dict(path=path, batch=_between(rng, 1, 32), tokens=_between(rng, 1, 511))
    kv_heads = rng.choice([1, 2, 4, 8, 12, 24, 40])
    dim, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 64, 128])
    dtype = rng.choice(["bf16", "f16"])
    batch = _between(rng, 1, 32)
    if path == "keep":
        tokens = _between(rng, 1, 63)
        return dict(path=path, batch=batch, tokens=tokens, length=_between(rng, 1, 600), ragged=rng.random() < 0.5,
                    kv_heads=min(8, kv_heads), dim=dim, page=page, accepted=rng.randint(1, min(tokens, 12)),
                    layers=_between(rng, 1, 40), dtype=dtype)
    group = rng.choice([1, 1, 2, 4, 5, 8])
    if path == "append":
        tokens = rng.choice([1, rng.randint(2, 64), _between(rng, 65, 24967)])
        while batch > 1 and batch * tokens > 24967:
            batch //= 2
        while kv_heads > 1 and batch * tokens * kv_heads * (group + 2) > 24967 * 40 * 3:
            kv_heads //= 2
        return dict(path=path, batch=batch, tokens=tokens, length=_between(rng, 1, 1600) - 1, ragged=rng.random() < 0.5,
                    heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page, rotary=rng.choice([dim, dim, dim // 2, dim // 4]),
                    layout=rng.choice(["half", "interleaved"]), counts=rng.random() < 0.3, dtype=dtype)
    kind = rng.choice(["step", "step", "draft", "draft", "draft", "chunk"])
    tokens = {"step": 1, "draft": rng.randint(2, 128), "chunk": _between(rng, 129, 4680)}[kind]
    mask = {"step": "causal", "draft": rng.choice(["tree", "tree", "tree", "causal"]), "chunk": rng.choice(["causal", "all"])}[kind]
    length = _between(rng, 1, 99840 if kind == "step" else 24960) - 1
    reads, products = 40 * 99840, 24 * 4680 * 24960
    while batch > 1 and batch * (length + tokens) * kv_heads > reads:
        batch //= 2
    while kv_heads > 1 and batch * (length + tokens) * kv_heads > reads:
        kv_heads //= 2
    while batch > 1 and batch * tokens * (length + tokens) * kv_heads * group > products:
        batch //= 2
    while group > 1 and batch * tokens * (length + tokens) * kv_heads * group > products:
        group //= 2
    while kv_heads > 1 and batch * tokens * (length + tokens) * kv_heads * group > products:
        kv_heads //= 2
    return dict(path=path, batch=batch, tokens=tokens, length=length, ragged=rng.random() < 0.5, heads=kv_heads * group,
                kv_heads=kv_heads, dim=dim, page=page, mask=mask, counts=rng.random() < 0.3, dtype=dtype)


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Settled tokens of every sequence: all alike, or spread evenly between about an eighth of the longest and the longest."""
    n, batch = case["length"], case["batch"]
    if not case["ragged"]:
        return [n] * batch
    return [max(0, n - (n * 7 // 8) * i // max(1, batch - 1) - (i % 3)) if i else n for i in range(batch)]


def _counts(case):
    """Pending tokens of every sequence: all, or some fewer, none in one of eight."""
    t, batch = case["tokens"], case["batch"]
    if not case["counts"]:
        return [t] * batch
    return [0 if i % 8 == 5 else max(1, t - i % 3) for i in range(batch)]


def _rope(rows, rotary, device):
    """cos and sin of position times frequency, fp32 [rows, rotary/2, 2]."""
    freq = 10000.0 ** (-torch.arange(rotary // 2, dtype=torch.float64) * 2 / rotary)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], -1).to(torch.float32).to(device)


def _parents(batch, tokens, gen, device):
    """Trees in level order: a node's parent comes before it, and parents never step back; the first nodes may all hang on
    the last settled token."""
    node = torch.arange(tokens, device=device)
    drawn = (torch.rand(batch, tokens, generator=gen, device=device) * node * 0.7).floor().long() - 1
    return torch.minimum(drawn.cummax(-1)[0], node - 1).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"

    def normal(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    b, t = case["batch"], case["tokens"]
    if case["path"] == "tree":
        return dict(case=case, parents=_parents(b, t, gen, dev))
    h, d, page, dtype = case["kv_heads"], case["dim"], case["page"], TYPES[case["dtype"]]
    lengths = _lengths(case)
    # every sequence's pages are scattered over the pool, behind them entries that name none; some pages are nobody's
    held = [-(-(n + t) // page) for n in lengths]
    total = sum(held) + 3
    pages = torch.rand(total, generator=gen, device=dev).argsort().to(torch.int32)
    table = torch.full((b, max(held) + 1), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = pages[at:at + n]
        at += n
    state = dict(case=case, table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device=dev))
    if case["path"] == "keep":
        layers, accepted = case["layers"], case["accepted"]
        state["k_pages"] = normal(layers, total, h, page, d, dtype=dtype)
        state["v_pages"] = normal(layers, total, h, page, d, dtype=dtype)
        # accepted nodes in order: the first, one after another as long as the draft's first guesses held, then ones of
        # further branches, which lie behind the places that they move to
        path, counts = torch.zeros(b, accepted, dtype=torch.int64), []
        host = torch.Generator().manual_seed(seed)
        for i in range(b):
            plain = int(torch.randint(1, accepted + 1, (1,), generator=host))
            plain = max(plain, 2 * accepted - t)
            others = torch.randperm(t - accepted, generator=host)[:accepted - plain].sort()[0] + accepted
            path[i] = torch.cat([torch.arange(plain), others])
            counts.append(int(torch.randint(1, accepted + 1, (1,), generator=host)))
        state["path"] = path.to(torch.int32).to(dev)
        state["counts"] = torch.tensor(counts, dtype=torch.int32, device=dev)
    else:
        heads = case["heads"]
        state["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=dev) if case["counts"] else None
        # keys whose channels differ in size, as attention layers have them
        size = torch.exp(0.5 * normal(1, h, 1, d))
        state["k_pages"] = torch.empty(total, h, page, d, dtype=dtype, device=dev)
        state["v_pages"] = torch.empty(total, h, page, d, dtype=dtype, device=dev)
        for i in range(0, total, 256):
            shape = state["k_pages"][i:i + 256].shape
            state["k_pages"][i:i + 256] = (normal(*shape) * size).to(dtype)
            state["v_pages"][i:i + 256] = normal(*shape).to(dtype)
        if case["path"] == "append":
            # the three are columns of one projection's rows
            qkv = normal(b, t, heads + 2 * h, d, dtype=dtype)
            state["q"], state["k"], state["v"] = qkv.split([heads, h, h], 2)
            state["positions"] = (state["lengths"][:, None] + torch.arange(t, device=dev)).to(torch.int32)
            state["rope"] = _rope(max(lengths) + t, case["rotary"], dev)
        else:
            state["q"] = normal(b, t, heads, d, dtype=dtype, std=1.5)
            if case["mask"] == "tree":
                state["parents"] = _parents(b, t, gen, dev)
                state["bits"] = _packed(_ancestors(state["parents"])[0])
    if own:
        from nanokv_b200.page_cache import PageCache, PageTable
        from nanokv_b200.rotary import Rotary
        state["pages"] = PageTable.over(table, state["lengths"], pages=total, page=page)
        if case["path"] == "keep":
            state["caches"] = [PageCache.over(state["pages"], k, v) for k, v in zip(state["k_pages"], state["v_pages"])]
        else:
            state["cache"] = PageCache.over(state["pages"], state["k_pages"], state["v_pages"])
        if case["path"] == "append":
            state["rotary"] = Rotary.over(state["rope"], head_dim=d, layout=case["layout"])
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return {"append": _append, "attend": _attend, "keep": _keep, "tree": _tree}[case["path"]](case, state)


def _places(state, tokens):
    """Page and row of tokens [batch, .], pages past the table or named by no entry taken as page 0."""
    page, table = state["case"]["page"], state["table"]
    entry = (tokens // page).clamp(0, table.shape[1] - 1)
    return table.gather(1, entry).clamp(min=0).long(), tokens % page


def _rotated(x, table, positions, layout):
    rd = 2 * table.shape[1]
    entry = table[positions.long()][:, :, None]
    c, s = entry[..., 0], entry[..., 1]
    xf = x.float()
    turned = xf[..., :rd]
    if layout == "half":
        a, b = turned[..., :rd // 2], turned[..., rd // 2:]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([turned, xf[..., rd:]], -1).to(x.dtype)


def _append(case, state):
    if own:
        q = state["cache"].append(state["k"], state["v"], state["q"], counts=state["counts"], rotary=state["rotary"],
                                  positions=state["positions"])
        return q, state["k_pages"], state["v_pages"]
    q, k = (_rotated(state[n], state["rope"], state["positions"], case["layout"]) for n in "qk")
    t = torch.arange(case["tokens"], device=q.device)
    pages, rows = _places(state, state["lengths"].long()[:, None] + t)
    if state["counts"] is None:
        state["k_pages"][pages, :, rows] = k
        state["v_pages"][pages, :, rows] = state["v"]
    else:
        there = t < state["counts"][:, None]
        state["k_pages"][pages[there], :, rows[there]] = k[there]
        state["v_pages"][pages[there], :, rows[there]] = state["v"][there]
    return q, state["k_pages"], state["v_pages"]


def _attend(case, state):
    q, bits = state["q"], state.get("bits")
    if own:
        return state["cache"].attend(q, counts=state["counts"], tree=bits, causal=case["mask"] == "causal")
    b, t, heads, d = q.shape
    h, page, table = case["kv_heads"], case["page"], state["table"].clamp(min=0).long()
    group, n = heads // h, table.shape[1] * page
    k, v = (state[x][table].transpose(1, 2).flatten(2, 3).float() for x in ("k_pages", "v_pages"))
    rows = q.float().reshape(b, t, h, group, d).transpose(1, 2).reshape(b, h, t * group, d)
    s = rows @ k.transpose(-1, -2) / math.sqrt(d)
    length = state["lengths"].long()[:, None]
    count = torch.full_like(length, t) if state["counts"] is None else state["counts"].long()[:, None]
    token, query = torch.arange(n, device=q.device), torch.arange(t, device=q.device)
    pending = token - length                                        # [b, n]
    if case["mask"] == "tree":
        at = pending.clamp(0, t - 1)
        words = bits.gather(2, (at // 32)[:, None].expand(b, t, n))
        seen = (words >> (at % 32)[:, None]) & 1 == 1
    elif case["mask"] == "causal":
        seen = pending[:, None] <= query[:, None]
    else:
        seen = torch.ones(b, t, 1, dtype=torch.bool, device=q.device)
    seen = (seen & ((pending >= 0) & (pending < count))[:, None]) | (pending < 0)[:, None]
    seen = seen & (query < count)[..., None]
    s.masked_fill_(~seen.repeat_interleave(group, 1)[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    w = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    # what lies behind a sequence's tokens has no weight, whatever it is
    v = torch.where((pending < count)[:, None, :, None], v, 0.0)
    out = (w @ v) / torch.where(total == 0, 1.0, total)
    lse = (top + total.log()).squeeze(-1)

    def back(x):
        return x.reshape(b, h, t, group, *x.shape[3:]).transpose(1, 2).flatten(2, 3).contiguous()

    return back(out).to(q.dtype), back(lse)


def _keep(case, state):
    if own:
        from nanokv_b200 import page_cache
        page_cache.keep(state["caches"], state["path"], state["counts"])
        return state["k_pages"], state["v_pages"]
    length = state["lengths"].long()[:, None]
    to = torch.arange(case["accepted"], device=length.device).expand(case["batch"], -1)
    there = to < state["counts"][:, None]
    pages, rows = (x[there] for x in _places(state, length + state["path"]))
    new_pages, new_rows = (x[there] for x in _places(state, length + to))
    for pool in (state["k_pages"], state["v_pages"]):
        pool[:, new_pages, :, new_rows] = pool[:, pages, :, rows]
    return state["k_pages"], state["v_pages"]


def _ancestors(parents):
    """sees [b, t, t]: node j is node i or one of its ancestors; depth [b, t]: how many ancestors there are."""
    t = parents.shape[-1]
    node = torch.arange(t, device=parents.device)
    reach = ((parents[..., None] == node) | (node[:, None] == node)).float()
    step = 1
    while step < t:                      # paths of twice as many steps each time
        reach = ((reach @ reach) > 0).float()
        step *= 2
    sees = reach > 0
    return sees, sees.sum(-1).to(torch.int32) - 1


def _packed(sees):
    t = sees.shape[-1]
    padded = torch.nn.functional.pad(sees, (0, -t % 32)).unflatten(-1, (-1, 32)).long()
    words = (padded << torch.arange(32, device=sees.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _tree(case, state):
    if own:
        from nanokv_b200 import ops
        return ops.tree_mask(state["parents"])
    sees, depth = _ancestors(state["parents"])
    return _packed(sees), depth


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b, t = case["batch"], case["tokens"]
    if case["path"] == "tree":
        words = -(-t // 32)
        return {"bytes": 4 * b * t * (2 + words), "flops": b * t * words}
    h, d = case["kv_heads"], case["dim"]
    if case["path"] == "keep":
        rows = b * case["accepted"] * h * case["layers"]
        return {"bytes": 2 * 2 * 2 * rows * d // 2, "flops": 0}      # (about half of the rows lie where they belong)
    heads, lengths, counts = case["heads"], _lengths(case), _counts(case)
    if case["path"] == "append":
        new = sum(counts)
        return {"bytes": 2 * 2 * d * (b * t * heads + 2 * new * h) + b * t * (4 + 4 * case["rotary"]),
                "flops": 3 * case["rotary"] * (b * t * heads + new * h)}
    held = sum(n + c for n, c in zip(lengths, counts) if c)
    if case["mask"] == "all":
        seen = sum(c * (n + c) for n, c in zip(lengths, counts))
    elif case["mask"] == "causal":
        seen = sum(c * n + c * (c + 1) // 2 for n, c in zip(lengths, counts))
    else:
        seen = sum(c * n + c * max(1, int(math.log2(c + 1))) for n, c in zip(lengths, counts))
    return {"bytes": 2 * 2 * held * h * d + 2 * 2 * b * t * heads * d + 4 * b * t * heads, "flops": 4 * seen * heads * d}


# ------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "keep": _exact_keep, "tree": _exact_tree}[case["path"]](case, state)


def _exact_append(case, state):
    """The rotation as a product of complex numbers, tokens put into their pages sequence by sequence."""
    turn = torch.view_as_complex(state["rope"].double())[state["positions"].long()][:, :, None]
    rd, page = case["rotary"], case["page"]
    results = []
    for name in "qk":
        y = state[name].double().clone()
        first, second = ((slice(0, rd // 2), slice(rd // 2, rd)) if case["layout"] == "half"
                         else (slice(0, rd, 2), slice(1, rd, 2)))
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        results.append(y)
    q, k = results
    pools = [state["k_pages"].double(), state["v_pages"].double()]
    table = state["table"].tolist()
    for i, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        done = 0
        while done < c:
            entry, row = divmod(n + done, page)
            more = min(c - done, page - row)
            for pool, new in zip(pools, (k, state["v"])):
                pool[table[i][entry], :, row:row + more] = new[i, done:done + more].transpose(0, 1).double()
            done += more
    return (q, *pools)


def _exact_attend(case, state):
    q = state["q"].double()
    b, t, heads, d = q.shape
    h, group = case["kv_heads"], heads // case["kv_heads"]
    if b * heads > 2048:
        return None
    out = torch.zeros_like(q)
    lse = torch.full((b, t, heads), -math.inf, dtype=torch.float64, device=q.device)
    for i, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        if c == 0:
            continue
        allowed = torch.ones(c, n + c, dtype=torch.bool, device=q.device)
        if case["mask"] == "causal":
            allowed[:, n:] = torch.ones(c, c, dtype=torch.bool, device=q.device).tril()
        elif case["mask"] == "tree":
            sees = torch.zeros(c, c, dtype=torch.bool)
            for node, up in enumerate(state["parents"][i, :c].tolist()):
                if up >= 0:
                    sees[node] = sees[up]
                sees[node, node] = True
            allowed[:, n:] = sees.to(q.device)
        pages = state["table"][i, :-(-(n + c) // case["page"])].long()
        for j in range(h):
            k, v = (state[x][:, j].index_select(0, pages).reshape(-1, d)[:n + c].double() for x in ("k_pages", "v_pages"))
            for head in range(j * group, j * group + group):
                for a in range(0, c, 1024):
                    s = q[i, a:min(c, a + 1024), head] @ k.T * d ** -0.5
                    s = torch.where(allowed[a:a + 1024], s, -math.inf)
                    total = torch.logsumexp(s, -1)
                    out[i, a:min(c, a + 1024), head] = torch.exp(s - total[:, None]) @ v
                    lse[i, a:min(c, a + 1024), head] = total
    return out, lse


def _exact_keep(case, state):
    pools = [state["k_pages"].double(), state["v_pages"].double()]
    page, table, path = case["page"], state["table"].tolist(), state["path"].tolist()
    for i, (n, c) in enumerate(zip(_lengths(case), state["counts"].tolist())):
        for j in range(c):
            (e0, r0), (e1, r1) = divmod(n + path[i][j], page), divmod(n + j, page)
            for pool in pools:
                pool[:, table[i][e1], :, r1] = pool[:, table[i][e0], :, r0]
    return tuple(pools)


def _exact_tree(case, state):
    bits, depths = [], []
    for parents in state["parents"].tolist():
        words, depth = [], []
        for node, up in enumerate(parents):
            words.append((words[up] if up >= 0 else 0) | 1 << node)
            depth.append(depth[up] + 1 if up >= 0 else 0)
        width = -(-len(parents) // 32)
        bits.append([[(x >> 32 * w) & 0xFFFFFFFF for w in range(width)] for x in words])
        depths.append(depth)
    bits = torch.tensor(bits, dtype=torch.int64)
    return torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32), torch.tensor(depths, dtype=torch.int32)
