"""Pages that sequences share, on the host: forking, copying on write, truncating and compacting against a model that
holds every sequence's rows apart, and the refusals of the new entry points (no GPU)."""

import ctypes as C
import os

import numpy as np
import pytest
import torch

from draftkv import _lib, ops, shared
from draftkv.paged import BlockPoolExhausted
from draftkv.shared import PagePool, SharedKVCache

needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")


@pytest.fixture
def host(monkeypatch):
    """Page copies by indexing, so that a cache works on the CPU (all but its kernels)."""
    def copy(store, src, dst):
        assert len(set(dst.tolist())) == dst.numel() and not set(dst.tolist()) & set(src.tolist())
        store[dst.long()] = store[src.long()]
        return store

    monkeypatch.setattr(ops, "paged_copy", copy)


def write(c, s, layer, pos, value):
    """Row pos of sequence s, as the append kernel stores it, through the device's table."""
    H, D, bs = c.n_heads, c.d_head, c.block_size
    blk = c.store[int(c.d_tables[s, layer, pos // bs])]
    assert c.pools[0].refs[int(c.d_tables[s, layer, pos // bs]) // c.n_layers] == 1, "a write to a page that others hold"
    blk[: H * bs * D].view(H, bs, D)[:, pos % bs] = value
    blk[H * bs * D:].view(H, D, bs)[:, :, pos % bs] = -value


def check(c, rows):
    c.pools[0].check_invariants()
    held = np.bincount(c.pages[c.pages >= 0], minlength=c.n_blocks)
    assert np.array_equal(held, c.pools[0].refs)
    for s in range(c.batch):
        for L in range(c.n_layers):
            k, v, pos = c.read(L, s)
            assert k.shape[0] == len(rows[s]) and np.array_equal(pos, np.arange(len(rows[s])))
            want = np.array(rows[s], np.float32) + 0.5 * L
            assert np.array_equal(k[:, 0, 0], want) and np.array_equal(v[:, -1, -1], -want)
            n = int(c.n_pages[s])
            assert c.d_tables[s, L, :n].tolist() == [int(p) * c.n_layers + L for p in c.pages[s, :n]]
    # the groups are true
    g = c.groups
    c._sync_groups()
    first, shared_rows = g._host
    assert len(shared_rows) == c.batch
    for x, y in zip(first, first[1:]):
        n = shared_rows[x]
        for s in range(x, y):
            assert rows[s][:n] == rows[x][:n]
            assert c.pages[s, : -(-n // c.block_size)].tolist() == c.pages[x, : -(-n // c.block_size)].tolist()


@pytest.mark.parametrize("bs", [1, 3, 16])
@pytest.mark.parametrize("seed", range(4))
def test_random_histories(host, bs, seed):
    rng = np.random.default_rng(100 * bs + seed)
    c = SharedKVCache(2, 2, 3, bs, 400, batch=3, max_tokens=60, device="cpu")
    rows, token = [[], [], []], 0
    for step in range(60):
        op = rng.choice(["append", "append", "append", "fork", "truncate", "compact"])
        if op == "append":
            cnt = [int(min(rng.integers(0, 8), 60 - len(r))) for r in rows]
            c.reserve(cnt)
            for s, n in enumerate(cnt):
                for _ in range(n):
                    token += 1
                    for L in range(2):
                        write(c, s, L, len(rows[s]), token + 0.5 * L)
                    rows[s].append(token)
            c.commit(cnt)
        elif op == "fork":
            par = rng.integers(0, c.batch, rng.integers(1, 6) if rng.random() < 0.5 else c.batch)
            if rng.random() < 0.7:
                par = np.sort(par)
            table = c.d_tables
            same = len(par) == c.batch
            c.fork(par)
            assert (c.d_tables is table) == same
            rows = [list(rows[p]) for p in par]
        elif op == "truncate":
            cut = [int(rng.integers(0, len(r) + 1)) for r in rows]
            c.truncate(cut)
            rows = [r[:n] for r, n in zip(rows, cut)]
        else:
            n = c.compact(int(rng.integers(300, 500)) if rng.random() < 0.5 else None)
            assert n == c.blocks_in_use and (c.pages.max() < n)
        check(c, rows)
        fill = {}
        for s, r in enumerate(rows):
            for i in range(len(r)):
                fill[int(c.pages[s, i // bs]), i % bs] = 1
        want = 1.0 - len(fill) / (c.blocks_in_use * bs) if c.blocks_in_use else 0.0
        assert c.fragmentation() == pytest.approx(want)
    c.truncate(0)
    assert c.blocks_in_use == 0 and c.pools[0].n_free == c.n_blocks
    check(c, [[] for _ in rows])


def test_a_short_pool_changes_nothing(host):
    c = SharedKVCache(1, 1, 2, 4, 5, batch=1, device="cpu", max_tokens=100)
    c.reserve([6])
    c.commit([6])
    c.fork([0, 0, 0])          # two pages, the second open and of three
    before = c.pages.copy(), c.pools[0].refs.copy()
    with pytest.raises(BlockPoolExhausted, match="4 pages wanted, 3"):
        c.reserve([4, 4, 2])   # two copies of the open page and two new ones
    assert np.array_equal(before[0], c.pages) and np.array_equal(before[1], c.pools[0].refs)
    c.reserve([2, 2, 2])       # two copies
    assert c.pools[0].n_free == 1 and len(set(c.pages[:, 1].tolist())) == 3
    with pytest.raises(BlockPoolExhausted, match="max_tokens"):
        c.reserve([200, 0, 0])
    with pytest.raises(ValueError, match="5 pages|too few|are live"):
        c.compact(2)


def test_the_last_holder_keeps_the_page(host):
    c = SharedKVCache(1, 1, 2, 4, 8, batch=1, device="cpu")
    c.reserve([2])
    c.commit([2])
    c.fork([0, 0])
    p = int(c.pages[0, 0])
    c.reserve([0, 1])
    assert c.pages[0, 0] == p and c.pages[1, 0] != p
    q = int(c.pages[1, 0])
    c.reserve([1, 1])
    assert c.pages[0, 0] == p and c.pages[1, 0] == q and c.blocks_in_use == 2


def test_forks_of_uneven_layers(host):
    """Layers appended one by one, as append() does: a fork in between copies what any layer writes."""
    c = SharedKVCache(2, 1, 2, 4, 20, batch=1, device="cpu")
    c._ensure_capacity(0, 0, 10)
    c.n_tokens[0, 0] = 10
    c._ensure_capacity(0, 1, 1)
    c.n_tokens[0, 1] = 1
    c.fork([0, 0])
    assert c.groups.bounds() == (0, 0, 0, 0) or c._regroup
    c._sync_groups()
    assert c.groups._host == ([0, 2], [1, 1])
    c.reserve([1, 0])
    assert all(c.pages[0, i] != c.pages[1, i] for i in range(3)) and c.blocks_in_use == 6


def test_refusals(host):
    c = SharedKVCache(1, 1, 2, 4, 8, batch=2, device="cpu")
    for bad in ([], [2], [-1], [[0]], [0, 5]):
        with pytest.raises(ValueError, match="parents"):
            c.fork(bad)
    with pytest.raises(ValueError, match="8 bits"):
        SharedKVCache(1, 1, 64, 16, 8, torch.float8_e4m3fn, device="cpu")
    with pytest.raises(ValueError, match="multiple of 32"):
        SharedKVCache(1, 1, 64, 16, 8, device="cpu", unit_keys=48)
    with pytest.raises(ValueError, match="d_head"):
        SharedKVCache(1, 1, 129, 16, 8, device="cpu")
    with pytest.raises(ValueError, match="positive"):
        SharedKVCache(1, 1, 64, 16, 8, batch=0, device="cpu")
    p = PagePool(3, 4)
    b = p.allocate()
    p.free(b)
    with pytest.raises(RuntimeError, match="double free"):
        p.free(b)
    with pytest.raises(RuntimeError, match="double free"):
        p.free(3)


def test_groups_are_checked():
    G = lambda first, sh: ops.PrefixGroups(first, sh, "cpu")
    assert G([0, 2, 3], [5, 5, 7]).bounds() == (2, 2, 5, 7)
    assert G([1, 3], [0, 4, 4, 0]).bounds() == (1, 2, 0, 4)
    assert G([], [0, 0]).bounds() == (0, 0, 0, 0)
    for first, sh in (([0], [0]), ([0, 0], [0]), ([0, 3], [1, 1]), ([-1, 1], [1]), ([0, 2], [1, 2]), ([0, 1], [1, 1]),
                      ([0, 1], [-1]), ([0, 1], [1 << 31])):
        with pytest.raises(ValueError):
            G(first, sh)
    g = G([0, 2], [3, 3])
    with pytest.raises(ValueError, match="one value per sequence"):
        g.update([0, 1], [3])
    assert not g.update([0, 2], [3, 3]) and g.update([0, 2], [4, 4]) and g.mem.tolist() == [4, 4, 0, 2, 0]


def test_ops_refuse_cpu_tensors():
    x = torch.zeros(1, 2, 8)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.beam_select(x, torch.zeros(1, 2, dtype=torch.float64), 2)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.paged_copy(x, torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.shared_attention(_lib.Paged(), 0, x[None], torch.zeros(1, dtype=torch.int32), 4, 32, 32)


# ---------------------------------------------------------------- the C entries' checks, before any launch
FAKE = 4096   # an address that is never read: every call below is refused on the host


def refused(rc, text, code=-1):
    assert rc == code and text in _lib.lib().dkv_last_error().decode(), (rc, _lib.lib().dkv_last_error())


@needs_lib
def test_c_copy_refuses():
    f = _lib.lib().dkv_paged_copy
    refused(f(FAKE, -1, 64, FAKE, FAKE, 1, None), "negative")
    refused(f(FAKE, 4, 64, FAKE, FAKE, -1, None), "negative")
    refused(f(None, 4, 64, FAKE, FAKE, 1, None), "NULL")
    refused(f(FAKE, 4, 64, None, FAKE, 1, None), "NULL")
    assert f(None, 4, 64, None, None, 0, None) == 0 and f(None, 4, 0, None, None, 3, None) == 0


@needs_lib
def test_c_beam_select_refuses():
    L = _lib.lib()
    ok = dict(x=FAKE, dt=0, stride=100, p=1, b=2, v=100, s=FAKE, k=4, o=FAKE, q=FAKE, t=FAKE, w=FAKE, n=1 << 20)

    def call(**kw):
        a = dict(ok, **kw)
        return L.dkv_beam_select(a["x"], a["dt"], a["stride"], a["p"], a["b"], a["v"], a["s"], a["k"], a["o"], a["q"], a["t"],
                                 a["w"], a["n"], None)

    for kw, text in ((dict(k=0), "k must"), (dict(k=65), "k must"), (dict(b=0), "beams"), (dict(b=65, k=64), "4096"),
                     (dict(v=0), "vocab"), (dict(v=1048577, stride=1 << 21), "vocab"), (dict(p=-1), "prompts"),
                     (dict(p=40000), "65535"), (dict(dt=3), "dtype"), (dict(stride=99), "row_stride"), (dict(x=None), "NULL"),
                     (dict(t=None), "NULL")):
        refused(call(**kw), text)
    refused(call(n=8), "workspace", -3)
    refused(call(w=None), "workspace", -3)
    assert call(p=0) == 0
    assert L.dkv_beam_select_workspace(1, 2, 100, 0) == 0 and L.dkv_beam_select_workspace(0, 2, 100, 1) == 0


@needs_lib
def test_c_shared_attention_refuses():
    L = _lib.lib()
    cache = dict(pool=FAKE, block_table=FAKE, batch=2, n_layers=2, n_kv_heads=2, head_dim=64, block_size=16, max_blocks=8, dtype=1)
    groups = dict(first=FAKE, shared=FAKE, n_groups=1, max_members=2, min_shared=3, max_shared=3)
    ok = dict(layer=0, q=FAKE, dt=0, T=1, hq=4, start=FAKE, count=None, max_len=128, prefix=32, unit=32, out=FAKE, w=FAKE, n=1 << 24)

    def call(c={}, g={}, **kw):
        a = dict(ok, **kw)
        return L.dkv_shared_attention(C.byref(_lib.Paged(**dict(cache, **c))), C.byref(_lib.Groups(**dict(groups, **g))), a["layer"],
                                      a["q"], a["dt"], a["T"], a["hq"], a["start"], a["count"], a["max_len"], a["prefix"], a["unit"], a["out"],
                                      a["w"], a["n"], None)

    for c, g, kw, text in (
            (dict(dtype=2), {}, {}, "cache dtype"), (dict(head_dim=129), {}, {}, "head_dim"), (dict(head_dim=0), {}, {}, "head_dim"),
            (dict(batch=0), {}, {}, "cache shape"), (dict(block_size=0), {}, {}, "cache shape"), (dict(pool=None), {}, {}, "NULL"),
            (dict(max_blocks=1 << 27), {}, {}, "positions"), ({}, dict(n_groups=3), {}, "n_groups"),
            ({}, dict(n_groups=-1), {}, "n_groups"), ({}, dict(max_members=0), {}, "group bounds"),
            ({}, dict(min_shared=4), {}, "group bounds"), ({}, dict(min_shared=-1), {}, "group bounds"),
            ({}, dict(max_members=3), {}, "group bounds"), ({}, dict(first=None), {}, "NULL"), ({}, dict(shared=None), {}, "NULL"),
            ({}, {}, dict(layer=2), "layer"), ({}, {}, dict(layer=-1), "layer"), ({}, {}, dict(dt=2), "query dtype"),
            ({}, {}, dict(hq=3), "multiple"), ({}, {}, dict(hq=0), "multiple"), ({}, {}, dict(unit=48), "unit_keys"),
            ({}, {}, dict(unit=0), "unit_keys"), ({}, {}, dict(prefix=40), "prefix_keys"), ({}, {}, dict(prefix=-32), "prefix_keys"), ({}, {}, dict(max_len=0), "max_len"), ({}, {}, dict(T=-1), "rows"),
            ({}, {}, dict(T=1 << 29), "rows"), ({}, {}, dict(q=None), "NULL"), ({}, {}, dict(out=None), "NULL"),
            ({}, {}, dict(start=None), "NULL")):
        refused(call(c, g, **kw), text)
    refused(call(n=64), "workspace", -3)
    refused(call(w=None), "workspace", -3)
    assert call(T=0) == 0


@needs_lib
@pytest.mark.parametrize("keys", [65536 + 32, (1 << 31) - 32])
def test_pieces_are_bounded(keys):
    """A position and a piece's keys more stay within 32 bits: longer pieces are refused, by the cache and by the C entry."""
    for name in ("prefix_keys", "unit_keys", "chunk_keys"):
        with pytest.raises(ValueError, match="at most 65536"):
            SharedKVCache(1, 1, 64, 16, 8, device="cpu", **{name: keys})
    L = _lib.lib()
    cache = _lib.Paged(pool=FAKE, block_table=FAKE, batch=1, n_layers=1, n_kv_heads=1, head_dim=64, block_size=16, max_blocks=8, dtype=1)
    groups = _lib.Groups(first=FAKE, shared=FAKE, n_groups=1, max_members=1, min_shared=64, max_shared=64)
    for prefix, unit, text in ((keys, 32, "prefix_keys"), (32, keys, "unit_keys")):
        refused(L.dkv_shared_attention(C.byref(cache), C.byref(groups), 0, FAKE, 0, 1, 1, FAKE, None, 128, prefix, unit, FAKE, FAKE,
                                       1 << 24, None), text)
        assert L.dkv_shared_attention_workspace(C.byref(cache), C.byref(groups), 1, 1, 128, prefix, unit) == 0


def test_a_recorded_step_belongs_to_its_groups():
    """Two caches alike in every bound: what a graph was recorded with tells their groups' memory apart."""
    made = [SharedKVCache(1, 1, 2, 4, 8, batch=2, device="cpu") for _ in range(2)]
    assert made[0].graph_key()[1:] == made[1].graph_key()[1:] and made[0].graph_key() != made[1].graph_key()


def test_engine_refuses(monkeypatch):
    from draftkv.engine import DraftKVEngine

    class Model:
        vocab_size, kv_dtype, n_kv_heads = 10, torch.float8_e4m3fn, 2

    e = DraftKVEngine(Model())
    with pytest.raises(ValueError, match="n must"):
        e.generate_samples([[1]], 0, 4)
    for n in (0, 33):
        with pytest.raises(ValueError, match="n_beams"):
            e.generate_beams([[1]], n, 4)
    with pytest.raises(IndexError):
        e.generate_beams([[11]], 2, 4)
    with pytest.raises(ValueError, match="share a float32 or bfloat16"):
        e.generate_samples([[1, 2]], 2, 4)
    assert e.generate_samples([], 2, 4) == [] and e.generate_beams([], 2, 4) == []
