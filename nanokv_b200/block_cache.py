"""Keys and values in 8-bit blocks, for sequences that grow a token or a chunk at a time.

``cache.CompressedHistory`` holds chunks encoded with trained operators.  ``BlockCache`` needs none: every 64 tokens of a
sequence and kv head become a block of 8-bit codes with one scale for K and one for V; the tokens of the open block are
kept in 16 bits and quantised once, when the block is complete, so that a cache does not depend on how its tokens were
cut into calls.  Query heads may share kv heads; the sequences of a batch have lengths of their own.

Blocks are found through a table of slots per sequence and kv head.  Attention can accumulate the weight it gave to
every block, and ``evict`` frees the blocks with the least of it by editing the table: no code is moved or quantised
again, and every kv head keeps blocks of its own choice.

Lengths live on the host and change with the calls; all work is enqueued on the current stream.  Calls that change a cache
(``append``, ``evict``, ``rewind``, ``attend`` with its weights) have to be ordered by the caller where they are on
different streams, as with any tensor.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib, ops
from .ops import BLOCK
from .rotary import Rotary


class BlockCache:
    def __init__(self, batch: int, kv_heads: int, head_dim: int, capacity: int, *, dtype: torch.dtype = torch.bfloat16,
                 device="cuda"):
        """Room for ``capacity`` tokens (rounded up to blocks) of every sequence."""
        if min(batch, kv_heads, capacity) <= 0:
            raise ValueError(f"batch, kv_heads and capacity must be positive; got {batch}, {kv_heads}, {capacity}")
        blocks = -(-capacity // BLOCK)
        rows, device = (batch, kv_heads), torch.device(device)
        self._take(torch.empty(*rows, blocks, BLOCK, head_dim, dtype=torch.uint8, device=device),
                   torch.empty(*rows, blocks, head_dim, BLOCK, dtype=torch.uint8, device=device),
                   torch.empty(*rows, blocks, 2, dtype=torch.float32, device=device),
                   torch.arange(blocks, dtype=torch.int32, device=device).expand(*rows, blocks).contiguous(),
                   torch.empty(*rows, BLOCK, head_dim, dtype=dtype, device=device),
                   torch.empty(*rows, head_dim, BLOCK, dtype=dtype, device=device), [0] * batch, None)

    @classmethod
    def over(cls, k_codes, v_codes, scales, table, k_tail, v_tail, lengths, *, weights=None) -> "BlockCache":
        """A cache over arrays that exist already, laid out as ``nkv_block_cache`` says; they are used in place.
        Every row of ``table`` must be a permutation of the slots."""
        self = cls.__new__(cls)
        self._take(k_codes, v_codes, scales, table, k_tail, v_tail, lengths, weights)
        return self

    def _take(self, k_codes, v_codes, scales, table, k_tail, v_tail, lengths, weights) -> None:
        if k_codes.dim() != 5 or k_codes.shape[3] != BLOCK:
            raise ValueError(f"k_codes must be [batch, kv_heads, blocks, {BLOCK}, head_dim]")
        batch, kv_heads, blocks, _, head_dim = k_codes.shape
        if head_dim not in (64, 128):
            raise ValueError(f"heads must be 64 or 128 wide; got {head_dim}")
        if k_tail.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"a block cache holds bf16 or fp16 rows, not {k_tail.dtype}")
        if weights is None:
            weights = torch.zeros(batch, kv_heads, blocks, dtype=torch.float32, device=k_codes.device)
        rows = (batch, kv_heads)
        for name, t, shape, dtype in (
                ("k_codes", k_codes, (*rows, blocks, BLOCK, head_dim), torch.uint8),
                ("v_codes", v_codes, (*rows, blocks, head_dim, BLOCK), torch.uint8),
                ("scales", scales, (*rows, blocks, 2), torch.float32), ("table", table, (*rows, blocks), torch.int32),
                ("k_tail", k_tail, (*rows, BLOCK, head_dim), k_tail.dtype),
                ("v_tail", v_tail, (*rows, head_dim, BLOCK), k_tail.dtype),
                ("weights", weights, (*rows, blocks), torch.float32)):
            if tuple(t.shape) != shape or t.dtype != dtype:
                raise ValueError(f"{name} must be {dtype} {list(shape)}; got {t.dtype} {list(t.shape)}")
            if not t.is_contiguous() or t.device != k_codes.device:
                raise ValueError(f"{name} must be contiguous, on one device with the others")
        if not k_codes.is_cuda:
            raise RuntimeError("nanokv_b200 runs on CUDA tensors only (there is no CPU path)")
        self.batch, self.kv_heads, self.head_dim, self.blocks = batch, kv_heads, head_dim, blocks
        self.dtype, self.device = k_tail.dtype, k_codes.device
        self.k_codes, self.v_codes, self.scales, self.table = k_codes, v_codes, scales, table
        self.k_tail, self.v_tail, self.weights = k_tail, v_tail, weights
        lengths = [int(n) for n in lengths]
        if len(lengths) != batch:
            raise ValueError(f"lengths must name {batch} sequences; got {len(lengths)}")
        if any(not 0 <= n <= self.capacity for n in lengths):
            raise ValueError(f"lengths must lie in 0 .. {self.capacity}; got {lengths}")
        self._lengths = lengths
        # the token behind the last whose row is in 16 bits (those of its block ahead of it are, too): how far back a rewind can go
        self._tail = list(lengths)
        self._array = (ctypes.c_int32 * batch)(*lengths)   # the lengths as the library reads them
        self._refresh()

    def _refresh(self) -> None:
        self._struct = _lib.BlockCache(
            self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.scales.data_ptr(), self.table.data_ptr(),
            self.k_tail.data_ptr(), self.v_tail.data_ptr(), self._array, self.batch, self.kv_heads, self.head_dim,
            self.blocks, ops.dtype_code(self.dtype))

    # ------------------------------------------------------------------ bookkeeping
    @property
    def capacity(self) -> int:
        return self.blocks * BLOCK

    @property
    def lengths(self) -> list[int]:
        """Tokens that every sequence holds."""
        return list(self._lengths)

    def _set_lengths(self, lengths: list[int]) -> None:
        try:
            self._array[:] = lengths
        except TypeError:
            self._array[:] = self._lengths
            raise
        self._lengths = lengths

    def _rows_of(self, x: torch.Tensor, name: str) -> int:
        if x.dim() != 4 or x.shape[0] != self.batch or x.shape[3] != self.head_dim:
            raise ValueError(f"{name} must be [{self.batch}, tokens, heads, {self.head_dim}]; got {list(x.shape)}")
        if x.dtype != self.dtype:
            raise ValueError(f"{name} must be {self.dtype}, as the cache is; got {x.dtype}")
        if x.device != self.device:
            raise (ValueError if x.is_cuda else RuntimeError)(f"{name} is on {x.device}, the cache on {self.device}")
        return x.shape[1]

    # ------------------------------------------------------------------ tokens in and out
    def append(self, k: torch.Tensor, v: torch.Tensor, *, counts=None, rotary: Rotary | None = None,
               positions: torch.Tensor | None = None) -> None:
        """Tokens k, v [batch, tokens, kv_heads, head_dim] put behind every sequence; of sequence b the first ``counts[b]``
        (host integers; default: all).  ``rotary`` rotates the keys by ``positions`` i32 [batch, tokens] on the way in."""
        tokens = self._rows_of(k, "k")
        if self._rows_of(v, "v") != tokens or k.shape[2] != self.kv_heads or v.shape[2] != self.kv_heads:
            raise ValueError(f"k and v must share [{self.batch}, tokens, {self.kv_heads}, {self.head_dim}]; got "
                             f"{list(k.shape)} and {list(v.shape)}")
        rotation = None
        if rotary is not None:
            if rotary.head_dim != self.head_dim or rotary.table.device != self.device:
                raise ValueError(f"the rotation is for heads of {rotary.head_dim} on {rotary.table.device}")
            ops._check_positions(positions, self.batch, tokens, self.device)
            rotation = ops._turns(rotary.table, positions, rotary.layout)
        ints = ops._host_ints(counts, self.batch, "counts")
        with ops._On(self.device):
            ops.block_append(self._struct, k, v, counts=ints, rotation=rotation)
        added = [tokens] * self.batch if counts is None else list(counts)
        longer = [n + more for n, more in zip(self._lengths, added)]
        self._tail = [n if more and n % BLOCK else t for n, more, t in zip(longer, added, self._tail)]
        self._set_lengths(longer)

    def rewind(self, lengths) -> None:
        """Every sequence cut back to its first ``lengths[b]`` tokens, as after a draft that was not accepted.  A cut may fall
        between blocks, or among the rows that the open block's 16-bit store still holds; weights of blocks that
        are given up go back to zero."""
        lengths = list(lengths)
        if len(lengths) != self.batch:
            raise ValueError(f"lengths must name {self.batch} sequences; got {len(lengths)}")
        if lengths == self._lengths:
            return
        # (sequences mostly stand alike: each kind of cut is looked at once)
        for n, now, tail in dict.fromkeys(zip(lengths, self._lengths, self._tail)):
            if not 0 <= n <= now:
                raise ValueError(f"a sequence that holds {now} tokens cannot be cut to {n}")
            if n != now and n % BLOCK and not (n // BLOCK == tail // BLOCK and n <= tail):
                raise ValueError(f"a sequence cannot be cut to {n}: the rows of its block {n // BLOCK} are not in 16 bits any more")
        left, held = ([(n + BLOCK - 1) // BLOCK for n in some] for some in (lengths, self._lengths))
        self._set_lengths(lengths)
        if left != held:
            if min(left) == max(left):
                self.weights[:, :, left[0]:] = 0
            else:
                for b, n in enumerate(left):
                    if n < held[b]:
                        self.weights[b, :, n:] = 0
        # rows in 16 bits of tokens that are given up count no longer
        self._tail = [t if t <= n else (n if n % BLOCK else 0) for n, t in zip(lengths, self._tail)]

    def read(self, start: int, stop: int):
        """k, v [batch, stop - start, kv_heads, head_dim]: the values that the cache holds for tokens [start, stop), zero past
        a sequence's length; for callers with an attention of their own."""
        with ops._On(self.device):
            return ops.block_read(self._struct, start, stop, dtype=self.dtype, device=self.device)

    # ------------------------------------------------------------------ attention and eviction
    def attend(self, q: torch.Tensor, *, counts=None, causal: bool = True, scale: float | None = None,
               weights: torch.Tensor | None = None, status: torch.Tensor | None = None):
        """(O [batch, tokens, heads, head_dim], lse f32 [batch, tokens, heads]) of queries over what the cache holds.

        ``causal``: the last ``counts[b]`` (default: all) queries are the sequence's last tokens, and each sees the tokens up
        to its own; otherwise every query sees all.  ``weights`` f32 [batch, kv_heads, blocks], ``cache.weights`` above
        all: the attention given to every block, summed over the queries and heads of its group, is added to it.
        A query that sees nothing, or lies past ``counts[b]``, gets O = 0 and lse = -inf."""
        self._rows_of(q, "q")
        if weights is not None and (weights.dtype != torch.float32 or weights.device != self.device
                                    or tuple(weights.shape) != (self.batch, self.kv_heads, self.blocks)
                                    or not weights.is_contiguous()):
            raise ValueError(f"weights must be contiguous float32 [{self.batch}, {self.kv_heads}, {self.blocks}] on {self.device}")
        if status is not None:
            ops._require_cuda(status)
        with ops._On(self.device):
            return ops.block_attend(self._struct, q, counts=ops._host_ints(counts, self.batch, "counts"), causal=causal,
                                    scale=1.0 / math.sqrt(self.head_dim) if scale is None else scale, weights=weights,
                                    status=status)

    def evict(self, keep: int, *, sinks: int = 1, recent: int = 1) -> None:
        """At most ``keep`` full blocks left in every sequence: the first ``sinks`` and the last ``recent`` stay, of the others
        those that ``weights`` ranks highest for the kv head at hand; the open block stays as well."""
        full = [n // BLOCK for n in self._lengths]
        partial = [int(n % BLOCK > 0) for n in self._lengths]
        before = self.table, self.weights
        self.table, self.weights = ops.block_evict(*reversed(before), full, partial, keep=keep, sinks=sinks, recent=recent)
        # nobody else may hold them: their memory is not to be used again before this stream is past the call
        for t in before:
            t.record_stream(torch.cuda.current_stream(self.device))
        lengths = list(self._lengths)
        for b, n in enumerate(full):
            if n <= keep:
                continue
            # the rows in 16 bits move with the open block; those of a block that is complete are given up
            self._tail[b] = keep * BLOCK + self._tail[b] % BLOCK if self._tail[b] // BLOCK == n and partial[b] else 0
            lengths[b] = keep * BLOCK + lengths[b] % BLOCK
        self._set_lengths(lengths)
        self._refresh()
