"""Paged full (authoritative) KV cache on the GPU, with host block pools.

Reference: draftkv/paged.py:29-181. Same allocator semantics -- a LIFO free
list over ``range(n_blocks)`` (first block handed out is ``n_blocks - 1``, a
freed block is reused next), per-layer block tables, ``truncate`` frees whole
emptied blocks from the tail and keeps a partly filled tail block,
``BlockPoolExhausted`` instead of corruption, ``RuntimeError`` on a double
free. The block *contents* live in one device pool:

    pool[phys_block] = K [n_kv_heads][block_size][d_head]  ++  V [n_kv_heads][d_head][block_size]

A batched cache gives every sequence its own ``BlockPool`` over its own range
of physical blocks, so each sequence's block ids are exactly those of a
batch-1 reference run. Block tables are mirrored to the device (int32
``[batch][n_layers][max_blocks]``) once per forward, before the kernels read
them.

``dtype=torch.float8_e4m3fn`` holds the cache in 8 bits: blocks are coded with
a power-of-two scale per block and head once they are full, and the last
``tail_rows`` rows of a sequence are also kept in bf16. A query reads its own
block's rows in bf16 and the blocks before it in 8 bits, so its result does not
depend on how the rows came (a verify block, one by one, after a rollback):
greedy speculative decoding equals plain decoding over the same cache.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence

import numpy as np
import torch

from . import ops
from ._lib import DKV_BF16, DKV_F32, Paged, Paged8, lib


class BlockPoolExhausted(RuntimeError):
    """Raised instead of silently corrupting state when the pool runs dry (paged.py:29-31)."""


class BlockPool:
    """Fixed pool of KV blocks handed out and returned whole (paged.py:33-73)."""

    def __init__(self, n_blocks: int, block_size: int) -> None:
        self.n_blocks = n_blocks
        self.block_size = block_size
        self._stack = list(range(n_blocks))      # pop() from the end: LIFO
        self._live: set[int] = set()

    def allocate(self) -> int:
        if not self._stack:
            raise BlockPoolExhausted(f"all {self.n_blocks} blocks of size {self.block_size} are in use")
        b = self._stack.pop()
        self._live.add(b)
        return b

    def allocate_many(self, n: int) -> list:
        """n allocate() calls at once: the blocks in the order they would be
        handed out. Raises (allocating nothing) when fewer than n are free."""
        if n > len(self._stack):
            raise BlockPoolExhausted(f"{n} blocks wanted, {len(self._stack)} of {self.n_blocks} free")
        if n <= 0:
            return []
        got = self._stack[-n:][::-1]
        del self._stack[-n:]
        self._live.update(got)
        return got

    def free(self, block: int) -> None:
        if block not in self._live:
            raise RuntimeError(f"double free of block {block}")
        self._live.remove(block)
        self._stack.append(block)

    @property
    def n_free(self) -> int:
        return len(self._stack)

    @property
    def n_used(self) -> int:
        return len(self._live)

    def check_invariants(self) -> None:
        assert len(set(self._stack)) == len(self._stack), "duplicate in free list"
        assert not (set(self._stack) & self._live), "block both free and allocated"
        assert len(self._stack) + len(self._live) == self.n_blocks, "blocks leaked"


def _torch_dtype(dtype) -> torch.dtype:
    if dtype in (None, np.float32, torch.float32, "float32", "f32"):
        return torch.float32
    if dtype in (torch.bfloat16, "bfloat16", "bf16"):
        return torch.bfloat16
    if dtype in (torch.float8_e4m3fn, "float8_e4m3fn", "fp8"):
        return torch.float8_e4m3fn
    raise ValueError(f"unsupported cache dtype {dtype!r} (float32, bfloat16 or float8_e4m3fn)")


def _version(t: Optional[torch.Tensor]) -> int:
    """Counts the changes of a tensor in place (0 where torch does not: none, or an inference tensor)."""
    return 0 if t is None or t.is_inference() else t._version


def auto_chunk_keys(batch: int, n_heads: int, max_tokens: int) -> int:
    """Keys per chunk of the verify/decode attention kernel: about 1024
    chunks (four per CU) over the cache's capacity, a power of two in
    [2048, 8192]. A workgroup takes a whole chunk where enough of them fill
    the chip, and a run of the chunk's units where they do not. Measured on
    one MI355X (bf16, head_dim 128): at batch 32, ctx 32k, 8192-key chunks are
    2.5-4% faster than 2048; at batch 1, ctx 262k, 2048 is best. Verify and decode use the cache's one value, so their rows
    stay bit-identical whatever it is."""
    units = max(1.0, batch * n_heads * max_tokens / 1024.0)
    return int(min(8192, max(2048, 1 << int(round(math.log2(units))))))


def default_device() -> torch.device:
    if not torch.cuda.is_available():
        raise RuntimeError("draftkv needs a ROCm GPU (torch.cuda.is_available() is False)")
    return torch.device("cuda", torch.cuda.current_device())


class PagedKVCache:
    """The full cache, in device blocks, behind the reference cache protocol.

    ``PagedKVCache(n_layers, n_heads, d_head, block_size=16, n_blocks=512,
    dtype=np.float32)`` is the reference signature (n_heads = KV heads);
    ``batch``, ``max_tokens``, ``device`` and ``chunk_keys`` (the fixed key
    chunk of the attention kernel; by default ``auto_chunk_keys``) are
    additions. With ``dtype=torch.float8_e4m3fn`` block_size is 16, 32, 64 or
    128 and ``tail_rows`` (a multiple of 16, by default block_size + 112) rows
    per sequence stay in bf16: ``truncate`` to a position inside a block needs
    that block's rows among them, which any rollback by up to ``max_rollback``
    rows has.
    """

    def __init__(self, n_layers: int, n_heads: int, d_head: int, block_size: int = 16,
                 n_blocks: int = 512, dtype=np.float32, *, batch: int = 1,
                 max_tokens: Optional[int] = None, device=None, chunk_keys: Optional[int] = None,
                 tail_rows: Optional[int] = None) -> None:
        self.n_layers, self.n_heads, self.d_head = n_layers, n_heads, d_head
        self.block_size, self.n_blocks, self.batch = block_size, n_blocks, batch
        self.dtype = _torch_dtype(dtype)
        self.device = torch.device(device) if device is not None else default_device()
        self.max_tokens = max_tokens if max_tokens is not None else n_blocks * block_size
        self.chunk_keys = chunk_keys if chunk_keys is not None else auto_chunk_keys(batch, n_heads, self.max_tokens)
        self.max_blocks = -(-self.max_tokens // block_size)
        self.pools = [BlockPool(n_blocks, block_size) for _ in range(batch)]
        self.fp8 = self.dtype == torch.float8_e4m3fn
        if self.fp8:
            self._init_fp8(tail_rows)
        else:
            per_block = 2 * n_heads * block_size * d_head
            self.store = torch.empty((batch * n_blocks, per_block), dtype=self.dtype, device=self.device)
        self.tables = np.full((batch, n_layers, self.max_blocks), -1, np.int32)   # local ids
        self.table_len = np.zeros((batch, n_layers), np.int64)
        self.n_tokens = np.zeros((batch, n_layers), np.int64)
        self.d_tables = torch.full((batch, n_layers, self.max_blocks), 0, dtype=torch.int32, device=self.device)
        self._dirty: Optional[tuple[int, int]] = None   # [lo, hi) block-index range to upload

    # ------------------------------------------------------------ 8 bits
    def _init_fp8(self, tail_rows: Optional[int]) -> None:
        bs, H, D = self.block_size, self.n_heads, self.d_head
        if bs not in (16, 32, 64, 128):
            raise ValueError(f"an 8-bit cache's block_size is 16, 32, 64 or 128, got {bs}")
        if not 1 <= D <= 256:
            raise ValueError(f"an 8-bit cache's d_head is at most 256, got {D}")
        self.tail_rows = bs + 112 if tail_rows is None else int(tail_rows)
        if self.tail_rows % 16 or self.tail_rows < bs + 16:
            raise ValueError(f"tail_rows must be a multiple of 16, at least block_size + 16, got {self.tail_rows}")
        self.max_rollback = self.tail_rows - bs - 15
        self._row_bytes = int(lib().dkv_paged8_row_bytes(H, D))
        kw = dict(dtype=torch.uint8, device=self.device)
        self.store = torch.empty((self.batch * self.n_blocks, int(lib().dkv_paged8_block_bytes(H, D, bs))), **kw)
        self.tail = torch.empty((self.batch, self.n_layers, self.tail_rows, self._row_bytes), **kw)
        # rows of long appends, grown by need: of eager calls, and of captured ones, whose graphs keep theirs
        self.hot = torch.empty((self.batch, 0, self._row_bytes), **kw)
        self._graph_hot: list = []
        self._hot_of: dict = {}                    # captured or not: the append whose rows are there
        # an open block's rows whose places in the tail a long append took (0xff: none)
        shape = Paged8(batch=self.batch, n_layers=self.n_layers, n_kv_heads=H, head_dim=D, block_size=bs)
        self.held = torch.full((int(lib().dkv_paged8_held_bytes(shape)),), 255, **kw)
        # the first position whose bf16 row is still there, per (sequence, layer)
        self.tail_from = np.zeros((self.batch, self.n_layers), np.int64)

    def _here(self, *tensors: Optional[torch.Tensor]) -> None:
        for t in tensors:
            if t is not None and t.device != self.store.device:
                raise ValueError(f"a tensor on {t.device} for a cache on {self.store.device}")

    def _long(self, T: int) -> bool:
        """Whether an append of T rows is more than the tail holds beside an open block."""
        return (self.block_size + T + 14) // 16 * 16 > self.tail_rows

    def _append8(self, layer: int, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, count: Optional[torch.Tensor]) -> Paged8:
        """The append, with its rows in a buffer too where it is long; the descriptor for their attention. Captured
        appends have a buffer of their own: a replay must not change what an eager attend() reads."""
        T = k.shape[1]
        if not self._long(T):
            if self._hot_of:      # (its rows may lie over those of the long one)
                capturing = torch.cuda.is_current_stream_capturing()
                if self._hot_of.get(capturing, (None,))[0] == layer:
                    del self._hot_of[capturing]
            d = self.desc()
            ops.paged8_append(d, layer, k, v, start, count)
            return d
        capturing = torch.cuda.is_current_stream_capturing()
        self._hot_of.pop(capturing, None)
        need = int(lib().dkv_paged8_hot_rows(self.desc(), T))
        hot = self.hot if not capturing else self._graph_hot[-1] if self._graph_hot else None
        if hot is None or need > hot.shape[1]:
            if hot is not None and hot.numel() and not capturing:
                hot.record_stream(torch.cuda.current_stream(self.device))
            hot = torch.empty((self.batch, need, self._row_bytes), dtype=torch.uint8, device=self.device)
            if capturing:
                self._graph_hot.append(hot)
            else:
                self.hot = hot
        d = self.desc(hot)
        ops.paged8_append(d, layer, k, v, start, count)
        self._hot_of[capturing] = (layer, T, *((t, _version(t)) for t in (start, count)))
        return d

    def _hot_rows_of(self, layer: int, T: int, start: torch.Tensor, count: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
        """The buffer with the rows of that append, or None where it is not the one whose rows are there."""
        capturing = torch.cuda.is_current_stream_capturing()
        of = self._hot_of.get(capturing)
        if of is None or of[:2] != (layer, T):
            return None
        for (was, version), t in zip(of[2:], (start, count)):
            if was is None and t is None:
                continue
            view = was is not None and t is not None and (t.data_ptr(), t.shape, t.stride(), t.dtype) == \
                (was.data_ptr(), was.shape, was.stride(), was.dtype)
            if _version(was) != version or capturing and not view:
                return None
            if not view:          # another tensor with the same values (the host waits for them)
                a, b = (x if x is not None else torch.full_like(y, T) for x, y in ((was, t), (t, was)))
                if (a.shape, a.dtype, a.device) != (b.shape, b.dtype, b.device) or not torch.equal(a, b):
                    return None
        return self.hot if not capturing else self._graph_hot[-1]

    def _writing(self, counts: np.ndarray, layers) -> None:
        """counts [batch, ...] rows are about to be written to ``layers``: what the tail then lacks is gone whether they
        are committed or not (a forward that fails), but for the open block, which a long append keeps."""
        n = self.n_tokens[:, layers]
        gone = np.minimum(-(-(n + counts) // 16) * 16 - self.tail_rows, n // self.block_size * self.block_size)
        self.tail_from[:, layers] = np.maximum(self.tail_from[:, layers], np.where(counts > 0, gone, 0))

    def _written(self, end: np.ndarray, layers) -> None:
        """Rows up to end [batch, ...] are in ``layers``: the tail holds the last tail_rows (whole 16s) of them."""
        self.tail_from[:, layers] = np.maximum(self.tail_from[:, layers], -(-end // 16) * 16 - self.tail_rows)

    # ------------------------------------------------------------ descriptor
    def desc(self, hot: Optional[torch.Tensor] = None):
        if self.fp8:
            hot = self.hot if hot is None else hot
            return Paged8(self.store.data_ptr(), self.d_tables.data_ptr(), self.tail.data_ptr(), hot.data_ptr(),
                          self.batch, self.n_layers, self.n_heads, self.d_head, self.block_size, self.max_blocks,
                          self.tail_rows, hot.shape[1], self.held.data_ptr())
        return Paged(self.store.data_ptr(), self.d_tables.data_ptr(), self.batch, self.n_layers, self.n_heads,
                     self.d_head, self.block_size, self.max_blocks,
                     DKV_BF16 if self.dtype == torch.bfloat16 else DKV_F32)

    # ------------------------------------------------------------ allocation
    def _ensure_capacity(self, s: int, layer: int, extra: int) -> None:   # paged.py:112-117
        need = self.n_tokens[s, layer] + extra
        while self.table_len[s, layer] * self.block_size < need:
            idx = int(self.table_len[s, layer])
            if idx >= self.max_blocks:
                raise BlockPoolExhausted(f"sequence {s} exceeds max_tokens={self.max_tokens}")
            self.tables[s, layer, idx] = self.pools[s].allocate()
            self.table_len[s, layer] += 1
            lo, hi = self._dirty or (idx, idx + 1)
            self._dirty = (min(lo, idx), max(hi, idx + 1))

    def _make_room(self, s: int, n: int) -> None:
        """Hook before sequence s takes n blocks (a fixed pool raises when short)."""

    def reserve(self, counts: Sequence[int]) -> None:
        """Allocate blocks for ``counts[s]`` more tokens in every layer, layer by
        layer as the reference's per-layer appends would (each sequence's pool
        hands its blocks to layer 0 first, then layer 1, ...), and push the new
        table entries to the device. Vectorized over (sequence, layer): only the
        pairs that need a block are visited."""
        cnt = np.asarray(counts, np.int64).reshape(self.batch)
        grow = cnt > 0
        if not grow.any():
            return
        bs = self.block_size
        need = self.n_tokens + cnt[:, None]
        want = np.where(grow[:, None], np.maximum(-(-need // bs), self.table_len), self.table_len)
        if int(want.max()) > self.max_blocks:
            s = int(np.flatnonzero((want > self.max_blocks).any(axis=1))[0])
            raise BlockPoolExhausted(f"sequence {s} exceeds max_tokens={self.max_tokens}")
        add = want - self.table_len
        for s in np.flatnonzero(add.any(axis=1)):
            self._make_room(int(s), int(add[s].sum()))
            got = self.pools[s].allocate_many(int(add[s].sum()))
            i = 0
            for L in np.flatnonzero(add[s]):
                k, t0 = int(add[s, L]), int(self.table_len[s, L])
                self.tables[s, L, t0: t0 + k] = got[i: i + k]
                i += k
        if add.any():
            lo = int(self.table_len[add > 0].min())
            hi = int(want.max())
            dl, dh = self._dirty or (lo, hi)
            self._dirty = (min(dl, lo), max(dh, hi))
            self.table_len = want
        self._upload()

    def _upload(self) -> None:
        if self._dirty is None:
            return
        lo, hi = self._dirty
        phys = self.tables[:, :, lo:hi] + (np.arange(self.batch, dtype=np.int32) * self.n_blocks)[:, None, None]
        phys = np.where(self.tables[:, :, lo:hi] >= 0, phys, 0).astype(np.int32)
        self.d_tables[:, :, lo:hi].copy_(ops.to_device(phys, self.device))
        self._dirty = None

    # ------------------------------------------------------------ batched device ops
    def append_layer(self, layer: int, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor,
                     count: Optional[torch.Tensor] = None) -> None:
        """Write ``k, v`` [batch, T, heads, d_head] at positions start[s]..; blocks
        must have been reserved."""
        if self.fp8:
            self._here(k)
            self._append8(layer, k, v, start, count)
            return
        ops.paged_append(self.desc(), layer, k, v, start, count)

    def attend(self, layer: int, q: torch.Tensor, start: torch.Tensor, max_len: int,
               out: Optional[torch.Tensor] = None, count: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of q [batch, T, heads, d_head] at positions start[s]..;
        count: the rows appended this forward when not all T (see append_layer).
        An 8-bit cache takes the queries of the rows that were just appended
        (the same T, start and count), float32 or bfloat16; of more rows than
        its tail holds, only right after their append_layer(), both eager or
        both captured, with start and count unchanged (a captured pair with
        the same tensors)."""
        if self.fp8:
            self._here(q)
            T = q.shape[1]
            hot = self._hot_rows_of(layer, T, start, count) if self._long(T) else None
            if hot is None and self._long(T):
                raise ValueError(f"attend() of {T} rows must follow their append_layer(): layer {layer}'s bf16 rows from "
                                 "that start are not there")
            return ops.paged8_attention(self.desc(hot), layer, q, start, max_len, out, count)
        return ops.paged_attention(self.desc(), layer, q, start, max_len, self.chunk_keys, out, count)

    def append_attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor,
                      max_len: int, count: Optional[torch.Tensor] = None) -> torch.Tensor:
        """append_layer, then attend: one layer's share of a forward."""
        if self.fp8:
            self._here(k, q)
            if q.shape[1] != k.shape[1]:
                raise ValueError(f"append_attend(): {q.shape[1]} queries for {k.shape[1]} rows")
            d = self._append8(layer, k, v, start, count)
            return ops.paged8_attention(d, layer, q, start, max_len, None, count)
        self.append_layer(layer, k, v, start, count)
        return self.attend(layer, q, start, max_len, count=count)

    def read_rows(self, layer: int, first: torch.Tensor, length: torch.Tensor, T: int):
        """The values an 8-bit cache stands for: float32 k, v [batch, T, heads,
        d_head] of positions first[s] .. first[s] + T - 1 (int32 [batch], on
        the device); rows past length[s], the rows the sequence holds, are zero."""
        if not self.fp8:
            raise ValueError("read_rows() is the 8-bit cache's; use read()")
        self._here(first)
        return ops.paged8_read(self.desc(), layer, first, length, T)

    def commit(self, counts: Sequence[int]) -> None:
        """Record that ``counts[s]`` rows were appended to every layer."""
        cnt = np.asarray(counts, np.int64)[:, None]
        self.n_tokens += cnt
        if self.fp8:
            self._written(np.where(cnt > 0, self.n_tokens, 0), slice(None))

    # ------------------------------------------------------------ reference protocol (batch 1 view)
    def append(self, layer: int, k, v, pos) -> None:                  # paged.py:120-128
        """Reference-protocol append for sequence 0 (k, v: (T, heads, d_head))."""
        if self.batch != 1:
            raise ValueError("append() is the batch-1 protocol; use reserve/append_layer/commit")
        k = torch.as_tensor(np.asarray(k, np.float32) if not torch.is_tensor(k) else k, device=self.device)
        v = torch.as_tensor(np.asarray(v, np.float32) if not torch.is_tensor(v) else v, device=self.device)
        pos = np.asarray(pos).reshape(-1)
        T = k.shape[0]
        if T == 0:
            return
        start = int(self.n_tokens[0, layer])
        if not np.array_equal(pos, np.arange(start, start + T)):
            raise ValueError("the device cache stores positions contiguously from 0")
        self._ensure_capacity(0, layer, T)
        self._upload()
        st = torch.tensor([start], dtype=torch.int32, device=self.device)
        if self.fp8:
            self._writing(np.array([T]), layer)
        self.append_layer(layer, k.float().contiguous()[None], v.float().contiguous()[None], st)
        self.n_tokens[0, layer] += T
        if self.fp8:
            self._written(self.n_tokens[:, layer], layer)

    def read(self, layer: int, seq: int = 0):                          # paged.py:130-138
        n = int(self.n_tokens[seq, layer])
        if n == 0:
            z = np.zeros((0, self.n_heads, self.d_head), np.float32)
            return z, z.copy(), np.zeros(0, np.int64)
        H, D, bs = self.n_heads, self.d_head, self.block_size
        if self.fp8:   # the one sequence's part of the cache
            d = self.desc()
            d.batch = 1
            d.block_table += 4 * seq * self.n_layers * self.max_blocks
            d.tail += seq * self.tail[0].numel()
            d.held += seq * (self.held.numel() // self.batch)
            at = torch.tensor([0, n], dtype=torch.int32, device=self.device)
            k, v = ops.paged8_read(d, layer, at[:1], at[1:], n)
            return k[0].cpu().numpy(), v[0].cpu().numpy(), np.arange(n, dtype=np.int64)
        nb = -(-n // bs)
        phys = self.tables[seq, layer, :nb].astype(np.int64) + seq * self.n_blocks
        blocks = self.store[torch.from_numpy(phys).to(self.device)].float().cpu().numpy()
        kb = blocks[:, : H * bs * D].reshape(nb, H, bs, D).transpose(0, 2, 1, 3).reshape(nb * bs, H, D)
        vb = blocks[:, H * bs * D:].reshape(nb, H, D, bs).transpose(0, 3, 1, 2).reshape(nb * bs, H, D)
        return kb[:n].copy(), vb[:n].copy(), np.arange(n, dtype=np.int64)

    def note_attention(self, layer: int, probs) -> None:               # paged.py:140-141
        pass

    def truncate(self, n_pos) -> None:                                 # paged.py:144-162
        """Drop positions >= n_pos (an int for every sequence, or one per sequence)."""
        cut = np.broadcast_to(np.asarray(n_pos, np.int64), (self.batch,))
        keep = np.minimum(self.n_tokens, cut[:, None])
        changed = keep != self.n_tokens
        if not changed.any():
            return
        if self.fp8:
            lost = changed & (keep % self.block_size != 0) & (keep // self.block_size * self.block_size < self.tail_from)
            if lost.any():
                s, L = (int(x[0]) for x in np.nonzero(lost))
                raise ValueError(f"sequence {s}: cannot cut {int(self.n_tokens[s, L])} rows to {int(keep[s, L])}: the "
                                 f"bf16 rows of that block are gone (kept from {int(self.tail_from[s, L])} on; a multiple "
                                 f"of block_size {self.block_size}, or a larger tail_rows, can)")
            self.tail_from = np.where(changed, np.minimum(self.tail_from, keep), self.tail_from)
            self._hot_of.pop(False, None)
        self.n_tokens = np.where(changed, keep, self.n_tokens)
        need = np.where(changed, -(-keep // self.block_size), self.table_len)
        # emptied tail blocks go back per sequence, layer by layer, last first
        for s, L in zip(*np.nonzero(self.table_len > need)):
            for idx in range(int(self.table_len[s, L]) - 1, int(need[s, L]) - 1, -1):
                self.pools[s].free(int(self.tables[s, L, idx]))
                self.tables[s, L, idx] = -1
            self.table_len[s, L] = need[s, L]

    @property
    def block_table(self) -> list:
        """Sequence 0's per-layer block ids (reference attribute)."""
        return [self.tables[0, L, : self.table_len[0, L]].tolist() for L in range(self.n_layers)]

    @property
    def pool(self) -> BlockPool:
        """Sequence 0's block pool (the reference's single pool)."""
        return self.pools[0]

    @property
    def length(self) -> int:
        return int(self.n_tokens[0, 0])

    def lengths(self) -> np.ndarray:
        return self.n_tokens[:, 0].copy()

    @property
    def blocks_in_use(self) -> int:
        return sum(p.n_used for p in self.pools)

    def fragmentation(self) -> float:                                  # paged.py:172-176
        cap = self.blocks_in_use * self.block_size
        return 0.0 if cap == 0 else 1.0 - float(self.n_tokens.sum()) / cap


def plan_blocks_needed(ctx: int, n_layers: int, block_size: int) -> int:   # paged.py:179-181
    """Blocks a context of ``ctx`` tokens occupies across all layers."""
    return n_layers * (-(-ctx // block_size))
