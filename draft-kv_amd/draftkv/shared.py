"""The paged full cache of sequences that share pages: many continuations of one prompt.

The reference's caches belong to one sequence (draftkv/paged.py:76-181). Here the sequences of a batch take their pages
from one pool and may have pages in common: ``fork`` makes a new batch out of the sequences of the old one (several
continuations of one, in another order, some dropped) without moving a row, the first row written to a page that
others hold copies that page, and a page nobody holds any more is free. Attention reads what the sequences of a group
have in common once for all of them (``ops.shared_attention``).

A page is a block of ``block_size`` tokens of every layer: page p of the pool is the physical blocks p * n_layers ..
p * n_layers + n_layers - 1 of the store, one per layer, in PagedKVCache's layout. The device's block tables are
PagedKVCache's too, so the drafter mirror and the append take them as they are.
"""

from __future__ import annotations

import contextlib
import math
from typing import Optional, Sequence

import numpy as np
import torch

from . import ops
from .paged import BlockPool, BlockPoolExhausted, PagedKVCache, _torch_dtype, auto_chunk_keys, default_device


class PagePool(BlockPool):
    """A block pool whose blocks may have several holders (``refs``): a block is free when its last holder gives it back."""

    def __init__(self, n_blocks: int, block_size: int) -> None:
        super().__init__(n_blocks, block_size)
        self.refs = np.zeros(n_blocks, np.int64)

    def allocate(self) -> int:
        b = super().allocate()
        self.refs[b] = 1
        return b

    def allocate_many(self, n: int) -> list:
        got = super().allocate_many(n)
        self.refs[got] = 1
        return got

    def next(self, n: int) -> list:
        """The blocks that allocate_many(n) will hand out, 0 < n <= n_free."""
        return self._stack[-n:][::-1]

    def free(self, block: int) -> None:
        if not 0 <= block < self.n_blocks or self.refs[block] == 0:
            raise RuntimeError(f"double free of block {block}")
        self.refs[block] -= 1
        if self.refs[block] == 0:
            super().free(block)

    def recount(self, refs: np.ndarray) -> None:
        """Other holders of the live blocks: refs per block (0 frees it; blocks that are free stay so)."""
        gone = np.flatnonzero((self.refs > 0) & (refs == 0)).tolist()
        self.refs = np.where(self.refs > 0, refs, 0)
        self._live.difference_update(gone)
        self._stack.extend(gone)

    def check_invariants(self) -> None:
        super().check_invariants()
        assert set(np.flatnonzero(self.refs > 0).tolist()) == self._live, "holders of free blocks"


def auto_prefix_keys(keys: int, members: int, per: int, least: int) -> int:
    """Keys per piece of what groups share, a power of two in [least, 2048]; keys: those of all groups and heads, members:
    sequences of the largest group, per: query heads per KV head. The tokens of a call do not count: verify and decode must
    cut alike. A wave walks a piece for 32 rows, so a call takes the longer of a piece and of the pieces' share of the 1024
    SIMDs, and beside it writes and reads a state per row and piece, 75 of which take as long as a key of the walk (150 of
    a float32 cache's, whose products count as twice as long; at the rates of large products they take 2.6 times): the least
    of max(P, keys tiles / 1024) + keys rows / 75 P.
    Measured (us; pieces of 128, 256, 512, 1024 and 2048 keys; one token each, 32 / 8 heads of 128, bf16): 8 sequences on
    8k 23 / 27 / 37, on 16k 35 / 29 / 37; 32 on 32k 123 / 85 / 72 / 68; 16 on 130k 310 / 220 / 170 / 151 / 147; 8 x 4 on 4k
    43 / 36 / 40; five tokens, 32 on 4k 83 / 65 / 64 / 68; pieces of 64, 128 and 256: 4 on 500, 9 / 3 heads of 64, float32
    16 / 20 / 28. Of 56 such calls of one token its choice takes 1 % longer than the best power of two (23 % at most),
    of 18 with five tokens 8 % (20 %). It does not count how many workgroups a CU holds (one of a float32 cache with heads
    of 128, two of a bf16 one), and was not fitted to the former."""
    tiles = -(-members * per // 32)
    want = max(keys * tiles / 1024, math.sqrt(keys * members * per * least / (75 * 128)), 1)
    return int(min(2048, max(least, 1 << round(math.log2(want)))))


# Keys per unit of a sequence's own, and the least of a piece: a step of 32 takes longer with float32 products.
# (us, units of 64 and 128: 16 x 3 rows on 900 keys, 12 heads of 64, float32 18 / 22; 32 on 8k unshared, bf16 240 / 210)
UNIT_KEYS = {torch.float32: 64, torch.bfloat16: 128}


class SharedKVCache(PagedKVCache):
    """``PagedKVCache`` with pages that sequences share.

    ``n_blocks`` is the pages of the one pool, each ``block_size`` tokens of all layers. ``batch`` is the number of
    sequences at first (the prompts); ``fork`` changes it. float32 or bfloat16. The attention sums what
    a group shares in pieces of ``prefix_keys`` (by default chosen from the groups) and the rest in units of ``unit_keys``
    (multiples of 32): plain and drafted decoding over caches whose sequences share the same agree bit for
    bit. Inside ``filling()``, for prompts, that of float32 queries is PagedKVCache's, in chunks of ``chunk_keys``."""

    def __init__(self, n_layers: int, n_heads: int, d_head: int, block_size: int = 16, n_blocks: int = 512,
                 dtype=np.float32, *, batch: int = 1, max_tokens: Optional[int] = None, device=None,
                 chunk_keys: Optional[int] = None, prefix_keys: Optional[int] = None,
                 unit_keys: Optional[int] = None) -> None:
        self.dtype = _torch_dtype(dtype)
        if self.dtype == torch.float8_e4m3fn:
            raise ValueError("a cache in 8 bits does not share pages (its open blocks' rows are per sequence): float32 or bfloat16")
        if min(n_layers, n_heads, d_head, block_size, n_blocks, batch) < 1:
            raise ValueError("SharedKVCache: sizes must be positive")
        if d_head > 128:
            raise ValueError(f"SharedKVCache: d_head is at most 128, got {d_head}")
        self.n_layers, self.n_heads, self.d_head = n_layers, n_heads, d_head
        self.block_size, self.n_blocks, self.batch = block_size, n_blocks, batch
        self.device = torch.device(device) if device is not None else default_device()
        self.max_tokens = max_tokens if max_tokens is not None else n_blocks * block_size
        self.chunk_keys = chunk_keys if chunk_keys is not None else auto_chunk_keys(batch, n_heads, self.max_tokens)
        self.prefix_keys = prefix_keys             # None: auto_prefix_keys
        self.unit_keys = unit_keys if unit_keys is not None else UNIT_KEYS[self.dtype]
        for name in ("chunk_keys", "prefix_keys", "unit_keys"):
            n = getattr(self, name)
            if n is not None and (n < 32 or n % 32 or n > 65536):
                raise ValueError(f"{name} must be a multiple of 32, at most 65536, got {n}")
        self.max_blocks = -(-self.max_tokens // block_size)
        self.fp8 = False
        self.pools = [PagePool(n_blocks, block_size)]
        self.store = torch.empty((n_blocks * n_layers, 2 * n_heads * block_size * d_head), dtype=self.dtype, device=self.device)
        self.pages = np.full((batch, self.max_blocks), -1, np.int32)
        self.n_pages = np.zeros(batch, np.int64)
        self.n_tokens = np.zeros((batch, n_layers), np.int64)
        self.root = np.arange(batch)               # the sequence at first that each comes from
        self.d_tables = torch.zeros((batch, n_layers, self.max_blocks), dtype=torch.int32, device=self.device)
        self.groups = ops.PrefixGroups([], [0] * batch, self.device)
        self._regroup = False                      # groups are to be worked out anew
        self._filling = False
        self._shared_keys = 0                      # keys that groups share, of all groups and heads

    def _not_recorded(self, why: str) -> None:
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(why)

    def _put(self, a: np.ndarray) -> torch.Tensor:
        with ops._device(self.store.device):
            return ops.to_device(a, self.device)

    # ------------------------------------------------------------ pages
    def _set_pages(self, s: np.ndarray, i: np.ndarray, p: np.ndarray) -> None:
        """Table entries (sequence, index) -> page on the host and the device."""
        if len(s) == 0:
            return
        s, i, p = (np.asarray(x, np.int64) for x in (s, i, p))
        L = np.arange(self.n_layers)
        at = ((s[:, None] * self.n_layers + L) * self.max_blocks + i[:, None]).reshape(-1)
        ids = (p[:, None] * self.n_layers + L).reshape(-1).astype(np.int32)
        self.d_tables.view(-1).index_copy_(0, self._put(at), self._put(ids))
        self.pages[s, i] = p                       # (last: what comes before may find no memory)

    def _copy_pages(self, src, dst) -> None:
        if len(src) == 0:
            return
        ab = self._put(np.array([src, dst], np.int32))
        ops.paged_copy(self.store.view(self.n_blocks, -1), ab[0], ab[1])

    def _own(self, lo: np.ndarray, hi: np.ndarray) -> None:
        """Give every sequence s pages lo[s] .. hi[s] - 1 of its own: new ones past its last, copies of those that others
        hold too. Raises before anything changes when the pool, or memory, is short."""
        pool, refs, b = self.pools[0], self.pools[0].refs, self.batch
        write = hi > lo
        if int(hi[write].max(initial=0)) > self.max_blocks:
            s = int(np.flatnonzero(write & (hi > self.max_blocks))[0])
            raise BlockPoolExhausted(f"sequence {s} exceeds max_tokens={self.max_tokens}")
        new = np.where(write, np.maximum(hi - self.n_pages, 0), 0)
        there = np.where(write, np.minimum(hi, self.n_pages) - lo, 0)   # pages to write that exist
        shared = []                                                    # (sequence, index) of those that others hold too
        first = self.pages[np.arange(b), np.minimum(lo, self.max_blocks - 1)]
        for s in np.flatnonzero((there > 1) | ((there == 1) & (refs[first] > 1))):
            shared += [(int(s), i) for i in range(int(lo[s]), int(lo[s] + there[s])) if refs[self.pages[s, i]] > 1]
        writers: dict = {}
        for s, i in shared:
            p = int(self.pages[s, i])
            writers[p] = writers.get(p, 0) + 1
        need = int(new.sum()) + sum(min(n, int(refs[p]) - 1) for p, n in writers.items())
        if need == 0:
            return
        self._not_recorded("reserve() before a forward is recorded: pages are taken on the host")
        if need > pool.n_free:
            raise BlockPoolExhausted(f"{need} pages wanted, {pool.n_free} of {pool.n_blocks} free")
        s_, i_, src = [], [], []
        left = {p: int(refs[p]) for p in writers}  # holders
        for s, i in shared:
            p = int(self.pages[s, i])
            if left[p] > 1:                        # (the last holder keeps it)
                left[p] -= 1
                s_.append(s), i_.append(i), src.append(p)
        got = np.asarray(pool.next(need), np.int64)   # copies first; they are taken once the device's work is queued
        grow = np.flatnonzero(new)
        n = new[grow]
        index = np.arange(int(n.sum())) - np.repeat(np.cumsum(n) - n, n) + np.repeat(self.n_pages[grow], n)
        self._copy_pages(src, got[: len(src)])
        self._set_pages(np.concatenate([np.asarray(s_, np.int64), np.repeat(grow, n)]),
                        np.concatenate([np.asarray(i_, np.int64), index]), got)
        pool.allocate_many(need)
        for p in src:
            pool.free(p)
        self.n_pages[grow] += n
        self._regroup = self._regroup or bool(src)

    def reserve(self, counts: Sequence[int]) -> None:
        """Pages for ``counts[s]`` more tokens of every layer, of the sequence's own: new ones, and a copy of its open page
        where others hold that too."""
        cnt = np.asarray(counts, np.int64).reshape(self.batch)
        bs = self.block_size
        lo = self.n_tokens.min(1) // bs
        self._own(lo, np.where(cnt > 0, -(-(self.n_tokens.max(1) + cnt) // bs), lo))
        self._sync_groups()

    def _ensure_capacity(self, s: int, layer: int, extra: int) -> None:
        bs, n = self.block_size, int(self.n_tokens[s, layer])
        lo = np.zeros(self.batch, np.int64)
        hi = lo.copy()
        lo[s], hi[s] = n // bs, -(-(n + extra) // bs)
        self._own(lo, hi)

    def _upload(self) -> None:
        """(the tables are written where they change)"""

    def fork(self, parents: Sequence[int]) -> None:
        """A new batch: sequence i is what sequence parents[i] is now, sharing its pages. Sequences that are nobody's
        parent give theirs back. What the batch's size shaped (a mirror, start positions) is the caller's to remake."""
        par = np.asarray(parents, np.int64)
        if par.ndim != 1 or par.size == 0 or par.min() < 0 or par.max() >= self.batch:
            raise ValueError(f"fork(): parents must be sequences 0..{self.batch - 1}, got {parents!r}")
        if par.size == self.batch and np.array_equal(par, np.arange(self.batch)):
            return
        self._not_recorded("fork() cannot be recorded: pages change hands on the host")
        idx = self._put(par)
        tables = self.d_tables.index_select(0, idx)
        if par.size == self.batch:
            self.d_tables.copy_(tables)            # (recorded graphs hold its address)
        else:
            self.groups = ops.PrefixGroups([], [0] * par.size, self.device)   # (where memory is short nothing has changed yet)
            self.d_tables, self.batch = tables, par.size
        self.pages, self.n_pages = self.pages[par], self.n_pages[par]
        self.n_tokens, self.root = self.n_tokens[par], self.root[par]
        held = self.pages[self.pages >= 0]
        self.pools[0].recount(np.bincount(held, minlength=self.n_blocks))
        self._regroup = True

    def truncate(self, n_pos) -> None:
        """Drop positions >= n_pos (an int for every sequence, or one per sequence); pages that empty go back."""
        cut = np.broadcast_to(np.maximum(np.asarray(n_pos, np.int64), 0), (self.batch,))
        keep = np.minimum(self.n_tokens, cut[:, None])
        if np.array_equal(keep, self.n_tokens):
            return
        self.n_tokens = keep
        need = -(-keep.max(1) // self.block_size)
        for s in np.flatnonzero(self.n_pages > need):
            for i in range(int(self.n_pages[s]) - 1, int(need[s]) - 1, -1):
                self.pools[0].free(int(self.pages[s, i]))
                self.pages[s, i] = -1
            self.n_pages[s] = need[s]
        self._regroup = True

    def compact(self, n_blocks: Optional[int] = None) -> int:
        """Move the live pages to the front of the pool, and with ``n_blocks`` make it that many pages long (more, or
        fewer: at least the live ones). Returns the live pages. Where memory is short it raises and changes nothing (the
        old store and the new one are there at once)."""
        pool = self.pools[0]
        live = np.flatnonzero(pool.refs > 0)
        n = live.size
        if n_blocks is not None and n_blocks < max(n, 1):
            raise ValueError(f"compact(): {n} pages are live, {n_blocks} are too few")
        self._not_recorded("compact() cannot be recorded: pages change places on the host")
        size = self.n_blocks if n_blocks is None else n_blocks
        store = self.store
        if size != self.n_blocks:
            store = torch.empty((size * self.n_layers, store.shape[1]), dtype=self.dtype, device=self.device)
        move = live[live >= n]
        holes = np.setdiff1d(np.arange(n), live)
        self._copy_pages(move, holes)              # (to pages that nobody holds)
        if store is not self.store:
            store[: n * self.n_layers].copy_(self.store[: n * self.n_layers])
        to = np.arange(self.n_blocks, dtype=np.int32)
        to[move] = holes
        moved = np.isin(self.pages, move) & (self.pages >= 0)
        s, i = np.nonzero(moved)
        there = self._put(np.arange(self.max_blocks) < self.n_pages[:, None]) if size < self.n_blocks else None
        self._set_pages(s, i, to[self.pages[s, i]])
        if there is not None:                      # (entries past a sequence's pages: ids that may lie behind the new store)
            self.d_tables.mul_(there[:, None])
        refs = np.zeros(size, np.int64)
        refs[to[live]] = pool.refs[live]
        pool.refs, pool.n_blocks = refs, size
        pool._live = set(range(n))
        pool._stack = list(range(size - 1, n - 1, -1))     # the lowest next
        self.store, self.n_blocks = store, size
        return n

    # ------------------------------------------------------------ groups
    def _sync_groups(self) -> None:
        """The groups of sequences next to each other that come from one prompt, and the rows they all have in common."""
        if not self._regroup:
            return
        self._not_recorded("reserve() before a forward is recorded: the groups of sequences changed")
        b, bs = self.batch, self.block_size
        shared = [0] * b
        cuts = [0, *(np.flatnonzero(np.diff(self.root)) + 1).tolist(), b]
        for x, y in zip(cuts, cuts[1:]):
            n = int(self.n_pages[x:y].min())
            same = (self.pages[x + 1:y, :n] == self.pages[x, :n]).all(0) if y - x > 1 else np.zeros(0, bool)
            common = int(same.size if same.all() else same.argmin())
            rows = min(common * bs, int(self.n_tokens[x:y].min()))
            shared[x:y] = [rows] * (y - x)
        self.groups.update(cuts if any(shared) else [], shared)
        self._shared_keys = self.n_heads * sum(shared[x] for x in cuts[:-1])
        self._regroup = False

    def graph_key(self) -> tuple:
        """What a recorded forward over this cache depends on beside its buffers' addresses."""
        return (self.groups.mem.data_ptr(), *self.groups.bounds(), self._shared_keys, self.prefix_keys, self.unit_keys)

    def _piece(self, q: torch.Tensor) -> int:
        return self.prefix_keys or auto_prefix_keys(self._shared_keys, self.groups.max_members, q.shape[2] // self.n_heads or 1,
                                                    UNIT_KEYS[self.dtype])

    # ------------------------------------------------------------ device ops
    def append_layer(self, layer: int, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor,
                     count: Optional[torch.Tensor] = None) -> None:
        """As PagedKVCache's; the pages must have been reserved."""
        self._here(k, v, start, count)
        with ops._device(self.store.device):
            ops.paged_append(self.desc(), layer, k, v, start, count)

    @contextlib.contextmanager
    def filling(self):
        """The rows inside are those of prompts, before anything is shared: attention of float32 queries takes the kernel
        whose workgroups walk the keys of many rows (4096 of a prompt, 32 / 8 heads of 128: 381 us; in units 1190)."""
        self._filling = True
        try:
            yield self
        finally:
            self._filling = False

    def attend(self, layer: int, q: torch.Tensor, start: torch.Tensor, max_len: int,
               out: Optional[torch.Tensor] = None, count: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of q [batch, T, heads, d_head] (float32 or bfloat16; the result has its type) at positions
        start[s] .., with what the sequences share read once."""
        self._here(q)
        self._sync_groups()
        if self._filling and self.groups.n_groups == 0 and q.dtype == torch.float32:   # (that kernel takes no other)
            with ops._device(q.device):
                return ops.paged_attention(self.desc(), layer, q, start, max_len, self.chunk_keys, out, count)
        return ops.shared_attention(self.desc(), layer, q, start, max_len, self._piece(q), self.unit_keys, self.groups, out, count)

    # ------------------------------------------------------------ views
    def read(self, layer: int, seq: int = 0):
        n = int(self.n_tokens[seq, layer])
        if n == 0:
            z = np.zeros((0, self.n_heads, self.d_head), np.float32)
            return z, z.copy(), np.zeros(0, np.int64)
        H, D, bs = self.n_heads, self.d_head, self.block_size
        nb = -(-n // bs)
        ids = self.pages[seq, :nb].astype(np.int64) * self.n_layers + layer
        blocks = self.store[torch.from_numpy(ids).to(self.device)].float().cpu().numpy()
        kb = blocks[:, : H * bs * D].reshape(nb, H, bs, D).transpose(0, 2, 1, 3).reshape(nb * bs, H, D)
        vb = blocks[:, H * bs * D:].reshape(nb, H, D, bs).transpose(0, 3, 1, 2).reshape(nb * bs, H, D)
        return kb[:n].copy(), vb[:n].copy(), np.arange(n, dtype=np.int64)

    @property
    def block_table(self) -> list:
        """Sequence 0's physical blocks per layer."""
        p = self.pages[0, : self.n_pages[0]].astype(np.int64) * self.n_layers
        return [(p + L).tolist() for L in range(self.n_layers)]

    def fragmentation(self) -> float:
        """The share of the live pages' rows that hold none."""
        live = self.blocks_in_use
        if live == 0:
            return 0.0
        fill = np.zeros(self.n_blocks, np.int64)
        n = self.n_tokens.max(1)
        for s in range(self.batch):
            at = self.pages[s, : self.n_pages[s]]
            fill[at] = np.maximum(fill[at], np.clip(n[s] - self.block_size * np.arange(at.size), 0, self.block_size))
        return 1.0 - float(fill.sum()) / (live * self.block_size)
