"""Calls of the shared cache that fail, or whose leftovers a later call might meet, on the host (no GPU)."""

import numpy as np
import pytest
import torch

from draftkv import ops
from draftkv.shared import SharedKVCache


@pytest.fixture
def host(monkeypatch):
    """Page copies by indexing, so that a cache works on the CPU (all but its kernels)."""
    def copy(store, src, dst):
        store[dst.long()] = store[src.long()]
        return store

    monkeypatch.setattr(ops, "paged_copy", copy)


def made(layers=2, bs=4, pages=8, rows=(6, 5, 9)):
    """A cache of sequences with rows of their own, the second dropped: live pages with a hole before them."""
    c = SharedKVCache(layers, 1, 2, bs, pages, batch=len(rows), max_tokens=40, device="cpu")
    c.reserve(rows)
    c.commit(rows)
    c.store.copy_(torch.arange(c.store.numel(), dtype=torch.float32).view(c.store.shape))
    c.fork([0, 2])
    return c


def state(c):
    return [c.batch, c.n_blocks, c.store.shape[0], c.pages.copy(), c.n_pages.copy(), c.n_tokens.copy(), c.d_tables.clone(),
            list(c.pools[0]._stack), set(c.pools[0]._live), c.pools[0].refs.copy(), c.pools[0].n_blocks]


def same(a, b):
    return all(np.array_equal(x, y) if isinstance(x, np.ndarray) else torch.equal(x, y) if torch.is_tensor(x) else x == y
               for x, y in zip(a, b))


def works(c):
    """Forks, grows and reads as a cache does whose parts agree; every page that it hands out is in the store."""
    c.pools[0].check_invariants()
    assert c.store.shape[0] == c.n_blocks * c.n_layers and c.pools[0].refs.size == c.n_blocks == c.pools[0].n_blocks
    before = [c.read(1, s)[0] for s in range(c.batch)]
    c.fork([1, 1, 0])
    c.reserve([5, 0, 5])
    c.commit([5, 0, 5])
    assert c.pages.max() < c.n_blocks and int(c.d_tables.max()) < c.store.shape[0]
    for s, p in enumerate([1, 1, 0]):
        assert np.array_equal(c.read(1, s)[0][: len(before[p])], before[p])
    c.pools[0].check_invariants()


@pytest.mark.parametrize("pages", [40, 5, 6])
def test_a_compaction_without_memory_changes_nothing(host, monkeypatch, pages):
    c = made()
    was = state(c)

    def full(*a, **kw):
        raise torch.OutOfMemoryError("no memory")

    with monkeypatch.context() as m:
        m.setattr(torch, "empty", full)
        with pytest.raises(torch.OutOfMemoryError):
            c.compact(pages)
    assert same(state(c), was)
    works(c)
    assert c.compact(pages + 10) == c.blocks_in_use
    works(c)


@pytest.mark.parametrize("pages", [None, 7, 9, 30])
def test_tables_name_no_page_behind_a_pool_that_shrank(host, pages):
    """Entries past a sequence's pages hold ids of pages that it gave back: none lies outside the store."""
    c = made(pages=20, rows=(30, 30, 13))
    c.truncate([9, 13])
    assert int(c.d_tables.max()) > 9 * c.n_layers          # (of pages that were given back)
    n = c.compact(pages)
    assert n == c.blocks_in_use == 7
    assert int(c.d_tables.min()) >= 0 and int(c.d_tables.max()) < c.store.shape[0]
    for s in range(c.batch):
        for L in range(c.n_layers):
            assert c.d_tables[s, L, : c.n_pages[s]].tolist() == [int(p) * c.n_layers + L for p in c.pages[s, : c.n_pages[s]]]
    if pages is not None and pages < 20:
        c.compact(40)
    works(c)


class Short:
    """Uploads and new tensors that find no memory from the n-th on."""

    def __init__(self, m, n):
        self.left = n
        for where, name in ((ops, "to_device"), (torch, "zeros"), (ops, "paged_copy")):
            m.setattr(where, name, self.wrap(getattr(where, name)))

    def wrap(self, f):
        def call(*a, **kw):
            self.left -= 1
            if self.left < 0:
                raise torch.OutOfMemoryError("no memory")
            return f(*a, **kw)
        return call


@pytest.mark.parametrize("call", [lambda c: c.fork([1, 0, 1]), lambda c: c.fork([1, 0]), lambda c: c.fork([1, 1]), lambda c: c.reserve([3, 9]),
                                  lambda c: c.compact(5), lambda c: c.compact(33), lambda c: c.compact()],
                         ids=["fork to more", "fork the other way", "fork", "reserve", "compact to fewer", "compact to more", "compact"])
@pytest.mark.parametrize("shared", [False, True])
def test_no_memory_anywhere_in_a_call(host, monkeypatch, call, shared):
    """Wherever memory runs out, the cache is what it was, or what the call makes of it; the call again does what it would have done."""
    def fresh():
        c = made(pages=30)
        if shared:
            c.fork([1, 1])
        return c

    want = fresh()
    call(want)
    for n in range(20):
        c = fresh()
        was = state(c)
        rows = [c.read(1, s)[0] for s in range(c.batch)]
        with monkeypatch.context() as m:
            short = Short(m, n)
            try:
                call(c)
            except torch.OutOfMemoryError:
                failed = True
            else:
                failed = False
                assert short.left >= 0 and same(state(c), state(want))
                break
        now = state(c)
        c.pools[0].check_invariants()
        held = np.bincount(c.pages[c.pages >= 0], minlength=c.n_blocks)
        assert np.array_equal(held, c.pools[0].refs)
        assert now[0] == was[0] and now[1:3] == was[1:3] and c.d_tables.shape[0] == c.groups.batch == c.batch
        for s in range(c.batch):
            assert np.array_equal(c.read(1, s)[0], rows[s])
            assert c.d_tables[s, 1, : c.n_pages[s]].tolist() == [int(p) * c.n_layers + 1 for p in c.pages[s, : c.n_pages[s]]]
        call(c)
        for a, b in zip(state(c)[3:6], state(want)[3:6]):
            assert np.array_equal(a, b)
        c.reserve([0] * c.batch)
        assert c.groups.mem.tolist() == [*c.groups._host[1], *c.groups._host[0],
                                         *[0] * (c.batch + 1 - len(c.groups._host[0]))]
        works_any(c)
    assert n > 0 and not failed


def works_any(c):
    c.pools[0].check_invariants()
    before = [c.read(0, s)[0] for s in range(c.batch)]
    c.reserve([2] * c.batch)
    c.commit([2] * c.batch)
    for s in range(c.batch):
        assert np.array_equal(c.read(0, s)[0][: len(before[s])], before[s])
    c.pools[0].check_invariants()


def test_groups_that_were_not_written_are_written_again(monkeypatch):
    g = ops.PrefixGroups([0, 2], [3, 3], "cpu")
    with monkeypatch.context() as m:
        Short(m, 0)
        with pytest.raises(torch.OutOfMemoryError):
            g.update([0, 1, 2], [5, 7])
    assert g.bounds() == (1, 2, 3, 3) and g.mem.tolist() == [3, 3, 0, 2, 0]
    assert g.update([0, 1, 2], [5, 7]) and g.bounds() == (2, 1, 5, 7) and g.mem.tolist() == [5, 7, 0, 1, 2]


@pytest.mark.parametrize("dtype,name", [(torch.float32, "paged_attention"), (torch.bfloat16, "shared_attention")])
def test_queries_of_prompts_go_to_a_kernel_that_takes_them(monkeypatch, dtype, name):
    """The unshared kernel, which prompts take, has float32 queries alone."""
    c = SharedKVCache(1, 1, 2, 4, 8, batch=1, device="cpu")
    called = []
    for f in ("paged_attention", "shared_attention"):
        monkeypatch.setattr(ops, f, lambda *a, f=f: called.append(f))
    q, start = torch.zeros(1, 3, 1, 2, dtype=dtype), torch.zeros(1, dtype=torch.int32)
    with c.filling():
        c.attend(0, q, start, 3)
    assert called == [name]
    c.attend(0, q, start, 3)
    assert called == [name, "shared_attention"]
