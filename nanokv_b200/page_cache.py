"""Keys and values in 16-bit pages, for sequences whose next tokens may be drafted as a tree.

``BlockCache`` quantises a token with its block and cannot take it back afterwards.  ``PageCache`` keeps rows as they came, in
pages that all sequences take from one pool, and tells settled tokens from pending ones: ``append`` writes the pending tokens
of a step behind the settled ones, ``attend`` lets them see the settled ones and, by a mask, one another (a chain, or the branches of
a draft), ``keep`` moves the rows of the accepted branch to the front of them, and ``PageTable.advance`` settles those.  What is
not settled is overwritten by the next step.

Which pages a sequence holds, and how many tokens of it are settled, is device memory of one ``PageTable``, shared by the
caches of all layers: calls read it when they run, so that a step captured into a graph can be replayed while sequences
grow.  Only ``reserve`` and ``release``, which deal out pages, happen on the host.  All work is enqueued on the current stream; calls
that change a table or a cache have to be ordered by the caller where they are on different streams, as with any tensor.
"""
from __future__ import annotations

import math
import operator

import torch

from . import _lib, ops
from .rotary import Rotary


class PageTable:
    """The pages and lengths of ``batch`` sequences of up to ``capacity`` tokens, over a pool of ``pages`` of ``page`` tokens."""

    def __init__(self, batch: int, capacity: int, *, pages: int, page: int = 64, device="cuda"):
        if min(batch, capacity, pages) <= 0:
            raise ValueError(f"batch, capacity and pages must be positive; got {batch}, {capacity}, {pages}")
        if page not in ops.PAGES:
            raise ValueError(f"a page holds 16, 32, 64 or 128 tokens; got {page}")
        device = torch.device(device)
        self._take(torch.full((batch, -(-capacity // page)), -1, dtype=torch.int32, device=device),
                   torch.zeros(batch, dtype=torch.int32, device=device), pages, page)
        self._held = [[] for _ in range(batch)]
        self._free = list(range(pages - 1, -1, -1))

    @classmethod
    def over(cls, table: torch.Tensor, lengths: torch.Tensor, *, pages: int, page: int) -> "PageTable":
        """A table over arrays that exist already and are used in place: table i32 [batch, entries] (an entry outside
        0 .. pages - 1 names no page), lengths i32 [batch].  Its pages are dealt out by the caller."""
        self = cls.__new__(cls)
        self._take(table, lengths, pages, page)
        self._held = self._free = None
        return self

    def _take(self, table, lengths, pages, page) -> None:
        if page not in ops.PAGES:
            raise ValueError(f"a page holds 16, 32, 64 or 128 tokens; got {page}")
        if table.dim() != 2 or table.dtype != torch.int32 or table.numel() == 0 or not table.is_contiguous():
            raise ValueError(f"table must be contiguous int32 [batch, entries]; got {table.dtype} {list(table.shape)}")
        if lengths.dtype != torch.int32 or tuple(lengths.shape) != (table.shape[0],) or not lengths.is_contiguous():
            raise ValueError(f"lengths must be contiguous int32 [{table.shape[0]}]; got {lengths.dtype} {list(lengths.shape)}")
        if lengths.device != table.device:
            raise ValueError("table and lengths must be on one device")
        if not table.is_cuda:
            raise RuntimeError("nanokv_b200 runs on CUDA tensors only (there is no CPU path)")
        if pages <= 0:
            raise ValueError(f"a pool has at least one page; got {pages}")
        self.table, self.lengths, self.pages, self.page = table, lengths, int(pages), int(page)
        self.batch, self.device = table.shape[0], table.device
        self.status = ops._word(self.device)            # what calls report into (ops.check_status)
        if self.status is None:
            raise RuntimeError("the first table of a device is made outside a graph capture: its status word would be the graph's")

    @property
    def capacity(self) -> int:
        return self.table.shape[1] * self.page

    @property
    def free(self) -> int:
        """Pages that no sequence holds."""
        return len(self._own())

    def _own(self) -> list[int]:
        if self._free is None:
            raise RuntimeError("the pages of a table over existing arrays are dealt out by the caller")
        return self._free

    def reserve(self, tokens) -> None:
        """Pages for ``tokens[b]`` tokens in all (host integers), settled and pending, for every sequence; those that a sequence
        holds already stay.  Nothing changes where the pool cannot give all of them."""
        free = self._own()
        tokens = [operator.index(n) for n in tokens]
        if len(tokens) != self.batch:
            raise ValueError(f"tokens must name {self.batch} sequences; got {len(tokens)}")
        if any(not 0 <= n <= self.capacity for n in tokens):
            raise ValueError(f"a sequence has room for 0 .. {self.capacity} tokens; got {tokens}")
        more = [max(0, -(-n // self.page) - len(held)) for n, held in zip(tokens, self._held)]
        if sum(more) > len(free):
            raise RuntimeError(f"{sum(more)} pages are needed and {len(free)} are free")
        if sum(more) == 0:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("pages cannot be dealt out inside a graph capture: reserve them before")
        entries = [b * self.table.shape[1] + len(self._held[b]) + i for b, n in enumerate(more) for i in range(n)]
        taken = free[len(free) - len(entries):][::-1]
        with ops._On(self.device):
            pairs = ops.upload(torch.tensor([entries, taken], dtype=torch.int64), self.device)
            self.table.view(-1).index_copy_(0, pairs[0], pairs[1].to(torch.int32))
        del free[len(free) - len(entries):]
        at = 0
        for held, n in zip(self._held, more):
            held.extend(taken[at:at + n])
            at += n

    def release(self, sequence: int) -> None:
        """A sequence emptied: its pages go back to the pool."""
        free = self._own()
        sequence = int(operator.index(sequence))      # (True would index a tensor otherwise than a list)
        if not 0 <= sequence < self.batch:
            raise ValueError(f"there are sequences 0 .. {self.batch - 1}; got {sequence}")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("pages cannot be given back inside a graph capture")
        self.table[sequence].fill_(-1)
        self.lengths[sequence].fill_(0)
        free.extend(reversed(self._held[sequence]))
        self._held[sequence] = []

    def advance(self, counts: torch.Tensor | int) -> None:
        """The first ``counts[b]`` pending tokens of every sequence (int32 tensor on the device, or one number for all) are settled.
        Once for all layers, behind their ``attend`` and ``keep``."""
        if isinstance(counts, torch.Tensor):
            ops._device_ints(counts, (self.batch,), "counts", self.device)
        elif operator.index(counts) < 0:
            raise ValueError(f"counts must not be negative; got {counts}")
        self.lengths.add_(counts)


class PageCache:
    """The keys and values of one layer in the pages of ``table``."""

    def __init__(self, table: PageTable, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16):
        if kv_heads <= 0:
            raise ValueError(f"kv_heads must be positive; got {kv_heads}")
        shape = (table.pages, kv_heads, table.page, head_dim)
        self._take(table, *(torch.empty(shape, dtype=dtype, device=table.device) for _ in range(2)))

    @classmethod
    def over(cls, table: PageTable, k_pages: torch.Tensor, v_pages: torch.Tensor) -> "PageCache":
        """A cache over pages [pages, kv_heads, page, head_dim] that exist already; they are used in place."""
        self = cls.__new__(cls)
        self._take(table, k_pages, v_pages)
        return self

    def _take(self, table, k_pages, v_pages) -> None:
        if k_pages.dim() != 4 or k_pages.shape[0] != table.pages or k_pages.shape[2] != table.page:
            raise ValueError(f"k_pages must be [{table.pages}, kv_heads, {table.page}, head_dim]; got {list(k_pages.shape)}")
        if k_pages.shape[3] not in (64, 128):
            raise ValueError(f"heads must be 64 or 128 wide; got {k_pages.shape[3]}")
        if k_pages.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"a page cache holds bf16 or fp16 rows, not {k_pages.dtype}")
        if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
            raise ValueError(f"v_pages must be as k_pages, {k_pages.dtype} {list(k_pages.shape)}; got {v_pages.dtype} {list(v_pages.shape)}")
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            if not t.is_contiguous() or t.device != table.device:
                raise ValueError(f"{name} must be contiguous, on the table's device")
        self.table, self.k_pages, self.v_pages = table, k_pages, v_pages
        self.kv_heads, self.head_dim, self.dtype, self.device = k_pages.shape[1], k_pages.shape[3], k_pages.dtype, table.device
        self._scale, self._scratch = 1.0 / math.sqrt(self.head_dim), {}     # scratch bytes by query heads and tokens
        self._struct = _lib.PageCache(k_pages.data_ptr(), v_pages.data_ptr(), table.table.data_ptr(), table.lengths.data_ptr(),
                                      table.batch, table.table.shape[1], table.pages, table.page, self.kv_heads, self.head_dim,
                                      ops.dtype_code(self.dtype))
        self._image = bytes(self._struct)

    def _rows(self, x: torch.Tensor, name: str) -> _lib.Tokens:
        return ops.page_rows(x, self._struct.batch, self.head_dim, self.dtype, self.device, name)

    def append(self, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None, *, counts: torch.Tensor | None = None,
               rotary: Rotary | None = None, positions: torch.Tensor | None = None) -> torch.Tensor | None:
        """Pending tokens k, v [batch, tokens, kv_heads, head_dim] written behind the settled ones, in place of what was pending;
        of sequence b the first ``counts[b]`` (int32 on the device; default: all).  ``rotary`` rotates the keys, and queries q [batch, tokens,
        heads, head_dim] with them, by ``positions`` i32 [batch, tokens]; default: the settled tokens' number and on, as for a chain.  Returns
        the rotated queries.  A token for which the table has no page is left out and reported (``ops.check_status``)."""
        rows, values, queries = self._rows(k, "k"), self._rows(v, "v"), None if q is None else self._rows(q, "q")
        tokens = k.shape[1]
        if v.shape[1] != tokens or rows.heads != self.kv_heads or values.heads != self.kv_heads:
            raise ValueError(f"k and v must share [{self.table.batch}, tokens, {self.kv_heads}, {self.head_dim}]; got "
                             f"{list(k.shape)} and {list(v.shape)}")
        if q is not None:
            if rotary is None:
                raise ValueError("queries are only rotated here: there is no rotation")
            if q.shape[1] != tokens:
                raise ValueError(f"there are {tokens} tokens of k and {q.shape[1]} of q")
        rotation = None
        if rotary is not None:
            if rotary.head_dim != self.head_dim or rotary.table.device != self.device:
                raise ValueError(f"the rotation is for heads of {rotary.head_dim} on {rotary.table.device}")
            if positions is not None:
                ops._check_positions(positions, self.table.batch, tokens, self.device)
            rotation = ops._turns(rotary.table, self.table.lengths if positions is None else positions, rotary.layout)
            if positions is None:
                rotation.positions = None
        with ops._On(self.device):
            out = None if q is None else q.new_empty(tuple(q.shape))
            ops.page_append(self._struct, rows, values, queries, out, tokens, counts=counts, rotation=rotation, device=self.device,
                            word=self.table.status.data_ptr())
        return out

    def attend(self, q: torch.Tensor, *, counts: torch.Tensor | None = None, tree: torch.Tensor | None = None, causal: bool = True,
               scale: float | None = None, status: torch.Tensor | None = None):
        """(O [batch, tokens, heads, head_dim], lse f32 [batch, tokens, heads]) of the pending tokens' queries over the settled
        tokens and one another, of sequence b the first ``counts[b]`` (int32 on the device; default: all).

        ``tree`` i32 [tokens, words] or [batch, tokens, words], as ``ops.tree_mask`` makes it: the pending tokens that each query
        sees, as bits.  Without it each sees those up to its own (``causal``) or all of them.  A query that sees nothing, or
        lies past ``counts[b]``, gets O = 0 and lse = -inf."""
        rows = self._rows(q, "q")
        if status is not None and (status.dtype != torch.int32 or status.device != self.device or status.numel() < 1):
            raise ValueError(f"status must be int32 on {self.device}")
        with ops._On(self.device):
            nbytes = self._scratch.get((rows.heads, q.shape[1]))
            if nbytes is None:
                nbytes = self._scratch[rows.heads, q.shape[1]] = ops.page_attend_workspace(self._struct, rows.heads, q.shape[1])
            return ops.page_attend(self._struct, q, rows, nbytes, counts=counts, tree=tree, causal=bool(causal),
                                   scale=self._scale if scale is None else float(scale),
                                   word=(self.table.status if status is None else status).data_ptr())

    def keep(self, path: torch.Tensor, counts: torch.Tensor | None = None) -> None:
        """``keep`` of this cache alone."""
        keep([self], path, counts)


def keep(caches, path: torch.Tensor, counts: torch.Tensor | None = None) -> None:
    """The accepted branch of a draft: the rows of pending tokens ``path`` i32 [batch, accepted] (ascending), of sequence b the first
    ``counts[b]`` (int32 on the device; default: all), moved to the front of the pending tokens in the caches of all layers, which
    share one ``PageTable``.  They are still pending: ``PageTable.advance(counts)`` settles them."""
    caches = list(caches)
    if not caches:
        return
    table = caches[0].table
    for cache in caches:
        if cache.table is not table:
            raise ValueError("the caches of a call share one PageTable")
    if path.dim() != 2 or path.device != table.device:
        raise ValueError(f"path must be int32 [{table.batch}, accepted] on {table.device}; got {list(path.shape)} on {path.device}")
    with ops._On(table.device):
        ops.page_keep([c._image for c in caches], table.batch, path, counts, word=table.status.data_ptr())
