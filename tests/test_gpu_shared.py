"""Many continuations of one prompt on the GPU: attention over pages that sequences share, page copies, beam selection and
the engine's calls that use them, against plain implementations in 64 bits.

Tolerances. u = 2^-24 is half a step of float32. A score is a float32 sum of up to 3 D products (each query in three bf16
parts, which leave u of it; D products for a float32 cache) of size at most top = max_k sum_d |q_d k_d| / sqrt(D): it is off
by (3 D + 4) u top, and 2^score-max by that, the difference's rounding (u of at most 2 top) and the instruction's 2 u. Sums
over the keys of a piece (at most `unit` of them) are chains of unit / 2 (l) and 3 unit (o, three parts of a probability)
additions, then unit / 32 rescalings and at most n / 32 pieces of the merge. So out is off by (2 (3 D + 8) top + 4 unit + n / 32 + 16) u times sum_k p_k |v_k|, numerator and
denominator each taking the scores' part once. bf16 queries: probabilities hold two bf16 parts (2^-16 of each), and the output is
rounded to bf16 (2^-8 of it).
"""

import math

import numpy as np
import pytest
import torch

from draftkv import ops
from draftkv._lib import DKV_BF16, DKV_F32, Paged

pytestmark = pytest.mark.gpu

F32, F64, BF16, I32 = torch.float32, torch.float64, torch.bfloat16, torch.int32
U = 2.0 ** -24


def i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def new_cache(batch, H, D, bs, most, dtype, unit, pages, layers=1):
    from draftkv import SharedKVCache
    c = SharedKVCache(layers, H, D, bs, pages, dtype, batch=batch, max_tokens=most, device="cuda", unit_keys=unit // 2 // 32 * 32 or 32,
                      prefix_keys=unit)
    c.store.fill_(math.nan)        # whatever no row was written to must not be seen
    return c


def tree(g, H, D, bs, dtype, unit, prompts, n, own, T, layers=1, layer=0):
    """A cache of prompts, each continued by n sequences with own[s] rows and T new ones, and the rows of every sequence:
    (cache, [k rows], [v rows], start)."""
    P = len(prompts)
    most = max(prompts) + max(own) + T
    pages = sum(-(-p // bs) for p in prompts) + P * n * (-(-(max(own) + T) // bs) + 1)
    c = new_cache(P, H, D, bs, most, dtype, unit, pages, layers)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    ck, cv = rnd(P, max(max(prompts), 1), H, D), rnd(P, max(max(prompts), 1), H, D)
    c.reserve(prompts)
    c.append_layer(layer, ck, cv, i32([0] * P), i32(prompts))
    c.commit(prompts)
    c.fork([p for p in range(P) for _ in range(n)])
    b = P * n
    new = [o + T for o in own]
    k, v = rnd(b, max(new), H, D), rnd(b, max(new), H, D)
    start = [prompts[s // n] for s in range(b)]
    c.reserve(new)
    c.append_layer(layer, k, v, i32(start), i32(new))
    c.commit(new)
    ks = [torch.cat([ck[s // n, :prompts[s // n]], k[s, :new[s]]]) for s in range(b)]
    vs = [torch.cat([cv[s // n, :prompts[s // n]], v[s, :new[s]]]) for s in range(b)]
    return c, ks, vs, [a + o for a, o in zip(start, own)]


def attention(q, k, v, last):
    """float64 attention of q [T, Hq, D] over rows k, v [n, H, D], row t over keys 0 .. last[t]: (out, sum p |v|, top)."""
    T, Hq, D = q.shape
    H = k.shape[1]
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    top = 0.0
    for t in range(T):
        n = last[t] + 1
        if n <= 0:
            continue
        for h in range(H):
            qq = q[t, h * (Hq // H):(h + 1) * (Hq // H)]
            w = torch.softmax(qq @ k[:n, h].t().contiguous() / math.sqrt(D), -1)
            out[t, h * (Hq // H):(h + 1) * (Hq // H)] = w @ v[:n, h]
            size[t, h * (Hq // H):(h + 1) * (Hq // H)] = w @ v[:n, h].abs()
            top = max(top, float((qq.abs() @ k[:n, h].abs().t().contiguous()).max()) / math.sqrt(D))
    return out, size, top


def bound(out, size, top, D, unit, n, qdtype, cache_dtype):
    e = (2 * (3 * D + 8) * top + 4 * unit + n / 32 + 16) * U
    if qdtype == BF16:
        e += 2.0 ** -16 if cache_dtype == BF16 else 0.0
        return e * size + 2.0 ** -8 * (out.abs() + e * size)
    return e * size


def attend(c, q, start, most, groups, layer=0, **kw):
    return ops.shared_attention(c.desc(), layer, q, i32(start), most, c.prefix_keys, c.unit_keys, groups, **kw)


# D, KV heads, query heads per KV head, block, cache, unit, prompts, continuations each, T
CASES = [
    (64, 3, 3, 16, F32, 64, [501], 4, 1), (64, 3, 3, 16, BF16, 128, [501], 4, 1), (128, 2, 4, 16, BF16, 128, [700, 33], 8, 1),
    (128, 2, 4, 16, F32, 64, [300], 5, 3), (128, 1, 4, 32, BF16, 256, [1030], 9, 5), (96, 2, 1, 16, BF16, 32, [65, 64, 63], 2, 2),
    (96, 1, 2, 48, F32, 32, [130], 3, 4), (32, 4, 2, 16, BF16, 96, [200], 3, 17), (32, 1, 8, 64, F32, 64, [129, 0, 1], 3, 9),
    (8, 2, 4, 16, F32, 32, [40], 6, 1), (8, 2, 4, 5, BF16, 32, [77], 3, 2), (40, 1, 3, 16, BF16, 64, [100], 3, 1),
    (1, 1, 1, 1, F32, 32, [5], 2, 1), (33, 2, 2, 7, F32, 64, [90, 12], 3, 3), (100, 1, 5, 16, BF16, 64, [150], 2, 6),
    (128, 1, 32, 16, BF16, 64, [90], 3, 2), (127, 1, 1, 16, F32, 32, [64], 2, 1), (16, 12, 1, 16, F32, 64, [900], 2, 3),
    (64, 1, 1, 128, BF16, 1024, [2000], 2, 40), (128, 2, 4, 16, BF16, 64, [31], 33, 1),
]


@pytest.mark.parametrize("qdtype", [F32, BF16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"d{c[0]}h{c[1]}x{c[2]}b{c[3]}{'f' if c[4] == F32 else 'h'}u{c[5]}p{c[6][0]}n{c[7]}t{c[8]}")
def test_attention(dev, case, qdtype):
    D, H, G, bs, dtype, unit, prompts, n, T = case
    g = torch.Generator(device=dev)
    g.manual_seed(D * 7 + n)
    own = [5 * s % 23 for s in range(len(prompts) * n)]
    c, ks, vs, start = tree(g, H, D, bs, dtype, unit, prompts, n, own, T)
    b = c.batch
    q = torch.randn(b, T, H * G, D, generator=g, device=dev).to(qdtype)
    out = c.attend(0, q, i32(start), max(s + T for s in start))
    assert out.dtype == qdtype and out.shape == q.shape
    for s in range(b):
        want, size, top = attention(q[s], ks[s], vs[s], [start[s] + t for t in range(T)])
        tol = bound(want, size, top, D, unit, start[s] + T, qdtype, dtype)
        err = (out[s].to(F64) - want).abs()
        assert (err <= tol).all(), (s, float((err / tol.clamp(min=1e-300)).max()))
        # the same without groups
        alone = attend(c, q, start, max(s + T for s in start), None)[s]
        assert ((alone.to(F64) - want).abs() <= tol).all(), s
    # the same bits with any bound on the lengths
    assert torch.equal(attend(c, q, start, c.max_blocks * bs, c.groups), out)


@pytest.mark.parametrize("qdtype", [F32, BF16])
@pytest.mark.parametrize("D,H,G,dtype,unit,ctx,n,T", [(128, 2, 4, BF16, 256, 2500, 6, 9), (64, 3, 3, F32, 128, 700, 8, 5),
                                                     (8, 2, 2, F32, 32, 100, 3, 4), (64, 1, 4, BF16, 128, 1290, 12, 17)])
def test_rows_do_not_depend_on_the_call(dev, D, H, G, dtype, unit, ctx, n, T, qdtype):
    """Bit for bit: all rows in one call, one row per call, and groups cut up; a sequence alone, with what it shared as what a
    group of one shares."""
    g = torch.Generator(device=dev)
    g.manual_seed(ctx)
    c, _, _, start = tree(g, H, D, 16, dtype, unit, [ctx], n, [3 * s for s in range(n)], T)
    q = torch.randn(n, T, H * G, D, generator=g, device=dev).to(qdtype)
    most = max(start) + T
    out = c.attend(0, q, i32(start), most)
    for t in range(T):
        one = c.attend(0, q[:, t:t + 1].contiguous(), i32([s + t for s in start]), most)
        assert torch.equal(one[:, 0], out[:, t]), t
    shared = c.groups._host[1][0]
    assert shared >= 64
    for s in range(n):
        d = c.desc()
        d.batch = 1
        d.block_table += 4 * s * c.n_layers * c.max_blocks
        one = ops.shared_attention(d, 0, q[s:s + 1].contiguous(), i32(start[s:s + 1]), start[s] + T, c.prefix_keys, c.unit_keys,
                                   ops.PrefixGroups([0, 1], [shared], dev))
        assert torch.equal(one[0], out[s]), s
    for first in ([0, 1, n], [0, n - 1, n], [0, 2, n], list(range(n + 1))):
        again = attend(c, q, start, most, ops.PrefixGroups(first, [shared] * n, dev))
        assert torch.equal(again, out), first
    # another division of the keys: other bits, and the same result whichever sequences have it
    for first, sh in (([1, n - 1], [0] + [shared - 1] * (n - 2) + [0]), ([0, n], [40] * n), ([0, 2, n], [0, 0] + [shared] * (n - 2))):
        again = attend(c, q, start, most, ops.PrefixGroups(first, sh, dev))
        for s in range(n):
            if sh[s] // 32 == shared // 32:
                assert torch.equal(again[s], out[s]), (first, s)
            if sh[s] == 0:
                assert torch.equal(again[s], attend(c, q, start, most, None)[s]), (first, s)


def test_many_rows_are_cut_into_launches(dev):
    """More rows than the workspace holds partials for: the same bits as in calls of a few."""
    g = torch.Generator(device=dev)
    g.manual_seed(5)
    H, G, D, unit, T = 2, 32, 128, 32, 260
    c, _, _, start = tree(g, H, D, 16, BF16, unit, [4000], 3, [0, 40, 80], T)
    from draftkv._lib import lib
    import ctypes
    assert lib().dkv_shared_attention_workspace(ctypes.byref(c.desc()), ctypes.byref(c.groups.desc()), T, H * G, max(start) + T,
                                                c.prefix_keys, c.unit_keys) < 600 << 20
    q = torch.randn(3, T, H * G, D, generator=g, device=dev)
    out = c.attend(0, q, i32(start), max(start) + T)
    for t in (0, 1, 100, 131, 200, 258):
        few = c.attend(0, q[:, t:t + 2].contiguous(), i32([s + t for s in start]), max(start) + T)
        assert torch.equal(few, out[:, t:t + 2]), t


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 20])
def test_counts_empty_sequences_and_values_that_are_not_finite(dev, D, dtype):
    """Padding rows see what the last one does, an empty sequence's are zero, and infinities or NaN in rows that a query
    must not see do not reach it, while they do reach those that see them."""
    H, G, unit, T, n, ctx = 2, 3, 32, 12, 5, 70
    g = torch.Generator(device=dev)
    g.manual_seed(D)
    c, ks, vs, start = tree(g, H, D, 16, dtype, unit, [ctx], n, [0, 4, 9, 2, 30], T)
    count = [T, 5, 0, T, 1]
    start[3], count[3] = 0, 0                      # (as the engine passes a sequence that is done)
    bad = {0: (start[0] + 4, math.inf), 1: (start[1] + 3, math.nan), 4: (start[4], -math.inf)}
    for s, (pos, x) in bad.items():
        blk = int(c.d_tables[s, 0, pos // 16])
        c.store[blk][H * 16 * D:].view(H, D, 16)[1, 3, pos % 16] = x     # V
        c.store[blk][: H * 16 * D].view(H, 16, D)[0, pos % 16, 2] = x    # K of the other head
        vs[s][pos, 1, 3] = x
        ks[s][pos, 0, 2] = x
    q = torch.randn(n, T, H * G, D, generator=g, device=dev)
    out = c.attend(0, q, i32(start), max(s + T for s in start), count=i32(count))
    for s in range(n):
        end = start[s] + count[s]
        last = [min(start[s] + t, end - 1) for t in range(T)]
        want, size, top = attention(q[s], ks[s][:end], vs[s][:end], last)
        got = out[s].to(F64)
        if end == 0:
            assert (got == 0).all()
            continue
        odd = ~torch.isfinite(want)
        if s in bad:
            assert odd.any() and not odd.all()
            assert (~torch.isfinite(got) == odd).all(), s
            v = want[:, G:, 3]                       # infinities keep their sign
            inf = torch.isinf(v)
            assert torch.equal(got[:, G:, 3][inf], v[inf])
        top = 12.0 * math.sqrt(D) if not math.isfinite(top) else top     # (|q k| of normal values, by their number)
        tol = bound(want, size, top, D, unit, end, F32, dtype)
        ok = (got - want).abs() <= tol
        assert ok[~odd].all(), s


def test_a_mask_that_leaves_nothing_of_a_unit(dev):
    """Rows of one tile whose units end apart, positions at unit and block borders, contexts of one key."""
    H, G, D, unit = 1, 1, 64, 32
    g = torch.Generator(device=dev)
    for ctx in (1, 15, 16, 31, 32, 33, 63, 64, 65, 96):
        g.manual_seed(ctx)
        own = [0, 1, 15, 16, 17, 31, 32, 33, 64]
        c, ks, vs, start = tree(g, H, D, 16, BF16, unit, [ctx], len(own), own, 2)
        q = torch.randn(len(own), 2, G, D, generator=g, device=dev)
        out = c.attend(0, q, i32(start), max(start) + 2)
        for s in range(len(own)):
            want, size, top = attention(q[s], ks[s], vs[s], [start[s], start[s] + 1])
            assert ((out[s].to(F64) - want).abs() <= bound(want, size, top, D, unit, start[s] + 2, F32, BF16)).all(), (ctx, s)


def test_a_bound_that_is_too_short_drops_pieces_only(dev):
    """max_len below what sequences hold: their rows see the keys up to the end of the piece or unit that it lies in."""
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    D, unit = 64, 64
    for groups, most, n in ((True, 100, 128), (True, 64, 64), (True, 1, 64), (True, 33, 64), (False, 100, 128), (False, 1, 32), (False, 33, 64), (True, 290, 320)):
        c, ks, vs, start = tree(g, 2, D, 16, BF16, unit, [300], 3, [51, 52, 53], 1)      # 288 shared keys, then units of 32
        assert c.groups.bounds() == (1, 3, 288, 288)
        q = torch.randn(3, 1, 4, D, generator=g, device=dev)
        out = attend(c, q, start, most, c.groups if groups else None)
        for s in range(3):
            want, size, top = attention(q[s], ks[s][:n], vs[s][:n], [n - 1])
            tol = bound(want, size, top, D, unit, n, F32, BF16)
            assert ((out[s].to(F64) - want).abs() <= tol).all(), (most, s)


def test_layers_and_streams_and_out(dev):
    """Another layer than the first, another stream than torch's own, a given output, a page pool that forks moved."""
    g = torch.Generator(device=dev)
    g.manual_seed(9)
    c, ks, vs, start = tree(g, 2, 64, 16, BF16, 64, [200, 50], 3, [1, 20, 3, 4, 5, 40], 2, layers=3, layer=2)
    q = torch.randn(6, 2, 8, 64, generator=g, device=dev)
    ref = c.attend(2, q, i32(start), 300)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(q)
    with torch.cuda.stream(st):
        got = c.attend(2, q, i32(start), 300, out=out)
    st.synchronize()
    assert got is out and torch.equal(out, ref)
    par = [4, 4, 0, 5, 2]
    c.fork(par)
    c.compact()
    again = c.attend(2, q[par].contiguous(), i32([start[p] for p in par]), 300)
    for s, p in enumerate(par):      # (other groups, so other pieces)
        want, size, top = attention(q[p], ks[p], vs[p], [start[p], start[p] + 1])
        for got in (again[s], ref[p]):
            assert ((got.to(F64) - want).abs() <= bound(want, size, top, 64, 64, start[p] + 2, F32, BF16)).all(), s
        k, v, _ = c.read(2, s)
        assert np.array_equal(k, ks[p].float().cpu().numpy()) and np.array_equal(v, vs[p].float().cpu().numpy())


def test_prompts_take_the_unshared_kernel_inside_filling_alone(dev):
    """Rows of prompts there are those of an ordinary cache bit for bit; outside, and once something is shared, a row is the
    same in a call of one and of many."""
    from draftkv import PagedKVCache
    g = torch.Generator(device=dev)
    g.manual_seed(8)
    n, H, D = 70, 2, 64
    q, k, v = (torch.randn(2, n, h, D, generator=g, device=dev) for h in (8, H, H))
    c = new_cache(2, H, D, 16, 100, BF16, 32, 30)
    c.reserve([n, n])
    with c.filling():
        out = c.append_attend(0, q, k, v, i32([0, 0]), n)
    p = PagedKVCache(1, H, D, 16, 10, BF16, batch=2, device=dev, chunk_keys=c.chunk_keys)
    p.reserve([n, n])
    assert torch.equal(out, p.append_attend(0, q, k, v, i32([0, 0]), n))
    out = c.attend(0, q, i32([0, 0]), n)
    one = torch.cat([c.attend(0, q[:, t:t + 1].contiguous(), i32([t, t]), n) for t in range(n)], 1)
    assert torch.equal(out, one)
    c.commit([n, n])
    c.fork([0, 0])
    rows = lambda: c.attend(0, q[:, :3].contiguous(), i32([n - 3] * 2), n)
    want = rows()
    with c.filling():
        assert torch.equal(rows(), want)


def test_far_pages_pass_32_bits(dev):
    """Pages behind 2^31 elements of the store."""
    H, D, bs = 8, 128, 16
    pages = (1 << 31) // (2 * H * bs * D) + 200
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    from draftkv import SharedKVCache
    c = SharedKVCache(1, H, D, bs, pages, BF16, max_tokens=1000, device=dev, unit_keys=64, prefix_keys=64)
    k, v = (torch.randn(1, 300, H, D, generator=g, device=dev).to(BF16) for _ in range(2))
    c.reserve([300])
    assert int(c.pages[0, 0]) == pages - 1
    c.append_layer(0, k, v, i32([0]))
    c.commit([300])
    c.fork([0, 0])
    c.reserve([1, 1])
    kn, vn = (torch.randn(2, 1, H, D, generator=g, device=dev).to(BF16) for _ in range(2))
    c.append_layer(0, kn, vn, i32([300, 300]))
    c.commit([1, 1])
    q = torch.randn(2, 1, 2 * H, D, generator=g, device=dev)
    out = c.attend(0, q, i32([300, 300]), 301)
    for s in range(2):
        want, size, top = attention(q[s], torch.cat([k[0], kn[s]]), torch.cat([v[0], vn[s]]), [300])
        assert ((out[s].to(F64) - want).abs() <= bound(want, size, top, D, 64, 301, F32, BF16)).all()


def test_a_recorded_step_follows_the_groups(dev):
    """A captured append and attention, replayed while rows are added, sequences forked and eager work runs in between."""
    H, G, D, unit, n = 2, 4, 64, 64, 4
    g = torch.Generator(device=dev)
    g.manual_seed(2)
    c, ks, vs, start = tree(g, H, D, 16, BF16, unit, [150], n, [0, 1, 2, 3], 1)
    q, k, v = (torch.randn(n, 1, h, D, generator=g, device=dev) for h in (H * G, H, H))
    at = i32([s + 1 for s in start])
    c.reserve([1] * n)
    ref = c.append_attend(0, q, k, v, at, c.max_tokens)
    torch.cuda.synchronize()
    key = c.graph_key()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.append_attend(0, q, k, v, at, c.max_tokens)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref)
    for step in range(4):
        par = [[0, 0, 2, 3], [3, 2, 1, 0], [1, 1, 1, 1], [0, 1, 2, 3]][step]
        c.fork(par)
        start = [start[p] for p in par]
        c.reserve([1] * n)
        assert c.graph_key() == key
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device=dev))
        at.copy_(i32([s + 1 for s in start]))
        graph.replay()
        got = out.clone()
        torch.randn(1000, device=dev).sum().item()
        ref = c.append_attend(0, q, k, v, at, max(start) + 2)
        assert torch.equal(got, ref), step


def test_pages_do_not_change_hands_while_a_graph_is_recorded(dev):
    c = new_cache(2, 2, 64, 16, 100, BF16, 32, 20)
    c.reserve([20, 20])
    c.commit([20, 20])
    c.fork([0, 0])
    g = ops.PrefixGroups([], [0, 0], dev)
    x, at = torch.zeros(4, device=dev), i32([19, 19])
    q = torch.zeros(2, 1, 4, 64, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: c.fork([1, 0]), lambda: c.compact(), lambda: c.reserve([9, 9]),
                     lambda: g.update([0, 2], [16, 16]), lambda: c.attend(0, q, at, 20)):
            with pytest.raises(RuntimeError, match="record"):
                call()
        x += 1
    graph.replay()
    c.reserve([9, 9])
    assert g.update([0, 2], [16, 16]) and x.tolist() == [1.0] * 4 and c.groups.bounds() == (1, 2, 16, 16)


def test_attention_refuses(dev):
    c = new_cache(2, 2, 64, 16, 100, BF16, 32, 20)
    c.reserve([10, 10])
    c.commit([10, 10])
    q = torch.randn(2, 1, 4, 64, device=dev)
    st = i32([9, 9])
    with pytest.raises(ValueError, match="does not match"):
        c.attend(0, q[:1].contiguous(), st, 10)
    with pytest.raises(ValueError, match="contiguous"):
        c.attend(0, torch.randn(2, 1, 4, 128, device=dev)[..., ::2], st, 10)
    with pytest.raises(ValueError, match="unsupported dtype"):
        c.attend(0, q.half(), st, 10)
    with pytest.raises(ValueError, match="one value per sequence"):
        c.attend(0, q, st[:1], 10)
    with pytest.raises(ValueError, match="one value per sequence"):
        c.attend(0, q, st, 10, count=i32([1]))
    with pytest.raises(ValueError, match="must be torch.int32"):
        c.attend(0, q, st.long(), 10)
    with pytest.raises(ValueError, match="out must"):
        c.attend(0, q, st, 10, out=torch.empty(2, 1, 4, 32, device=dev))
    with pytest.raises(ValueError, match="must be torch.float32"):
        c.attend(0, q, st, 10, out=torch.empty(2, 1, 4, 64, device=dev, dtype=BF16))
    with pytest.raises(ValueError, match="layer"):
        c.attend(1, q, st, 10)
    with pytest.raises(ValueError, match="multiple of KV heads"):
        c.attend(0, q[:, :, :3].contiguous(), st, 10)
    with pytest.raises(ValueError, match="max_len"):
        c.attend(0, q, st, 0)
    with pytest.raises(ValueError, match="groups of"):
        attend(c, q, [9, 9], 10, ops.PrefixGroups([], [0], dev))
    with pytest.raises(ValueError, match="prefix_keys"):
        ops.shared_attention(c.desc(), 0, q, st, 10, 33, 32)
    assert c.attend(0, q[:, :0].contiguous(), st, 10).shape == (2, 0, 4, 64)


# ---------------------------------------------------------------- page copies
@pytest.mark.parametrize("dtype,elems", [(torch.uint8, 1), (torch.uint8, 37), (torch.uint8, 4099), (BF16, 3), (BF16, 1001), (BF16, 40000),
                                         (F32, 1), (F32, 7), (F32, 1030), (F32, 300000), (torch.float8_e4m3fn, 64)])
def test_paged_copy(dev, dtype, elems):
    g = torch.Generator(device=dev)
    g.manual_seed(elems)
    for n, pairs in ((2, 1), (40, 13), (40, 0)):
        size = torch.empty((), dtype=dtype).element_size()
        store = torch.randint(0, 256, (n, elems * size), dtype=torch.uint8, device=dev, generator=g).view(dtype)
        perm = torch.randperm(n, device=dev, generator=g)
        dst = perm[:pairs].to(I32)
        src = perm[pairs:][torch.randint(0, n - pairs, (pairs,), device=dev, generator=g)].to(I32)
        want = store.view(torch.uint8).clone()
        want[dst.long()] = want[src.long()]
        assert ops.paged_copy(store, src, dst) is store
        assert torch.equal(store.view(torch.uint8), want)


def test_paged_copy_at_odd_addresses_and_ids(dev):
    """A store that starts off 16 bytes; ids outside it are skipped; a page onto itself stays."""
    for off in (1, 2, 4, 8):
        mem = torch.randint(0, 256, (off + 6 * 64,), dtype=torch.uint8, device=dev)
        store = mem[off:].view(6, 64)
        want = mem.clone()
        want[off + 64 * 4: off + 64 * 5] = want[off: off + 64]
        ops.paged_copy(store, i32([0, -1, 6, 2, 3, 2]), i32([4, 1, 1, 2, 6, -5]))
        assert torch.equal(mem, want), off


def test_paged_copy_past_32_bits(dev):
    store = torch.empty((5, 3 << 29), dtype=torch.uint8, device=dev)
    for i in range(5):
        store[i].fill_(i + 1)
    ops.paged_copy(store, i32([0, 4]), i32([3, 2]))
    for i, x in enumerate((1, 2, 5, 1, 5)):
        assert int(store[i].min()) == x == int(store[i].max())


def test_paged_copy_replayed(dev):
    store = torch.arange(8 * 4096, device=dev, dtype=F32).view(8, 4096)
    src, dst = i32([0, 1]), i32([5, 6])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_copy(store, src, dst)
    for step in range(3):
        store.copy_(torch.randn(8, 4096, device=dev))
        src.copy_(i32([step, 1 + step]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(store[5], store[step]) and torch.equal(store[6], store[1 + step])


def test_paged_copy_refuses(dev):
    store = torch.zeros(4, 8, device=dev)
    for src, dst, text in ((i32([0]), i32([1, 2]), "sources"), (i32([0]).long(), i32([1]), "int32"), (i32([[0]]), i32([1]), "dims"),
                           (i32([0]).cpu(), i32([1]), "GPU")):
        with pytest.raises(ValueError, match=text):
            ops.paged_copy(store, src, dst)
    with pytest.raises(ValueError, match="contiguous"):
        ops.paged_copy(store.t(), i32([0]), i32([1]))
    ops.paged_copy(torch.zeros(0, 8, device=dev), i32([0]), i32([1]))
    ops.paged_copy(torch.zeros(4, 0, device=dev), i32([0]), i32([1]))


# ---------------------------------------------------------------- beam selection
def select(x, cum, k):
    """The definition, in float64: scores, beams and tokens [prompts, k]."""
    P, B, V = x.shape
    out = np.full((P, k), -np.inf), np.full((P, k), -1), np.full((P, k), -1)
    for p in range(P):
        cand = []
        for b in range(B):
            row = x[p, b].astype(np.float64)
            if np.isnan(row).any() or (row == np.inf).any() or not (row > -np.inf).any() or not cum[p, b] > -np.inf:
                continue
            m = row.max()
            lse = m + math.log(math.fsum(np.exp(row[row > -np.inf] - m)))
            best = np.argsort(-row, kind="stable")[:k]
            cand += [(-(cum[p, b] + (row[v] - lse)), b, -row[v], v) for v in best if row[v] > -np.inf]
        for j, (s, b, _, v) in enumerate(sorted(cand)[:k]):
            out[0][p, j], out[1][p, j], out[2][p, j] = -s, b, v
    return out


def check_select(x, cum, k, dev, dtype=F32):
    xd = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(dev).to(dtype)
    x = xd.float().cpu().numpy()
    s, b, v = (t.cpu().numpy() for t in ops.beam_select(xd, torch.from_numpy(np.ascontiguousarray(cum, np.float64)).to(dev), k))
    ws, wb, wv = select(x, cum, k)
    assert np.array_equal(b, wb) and np.array_equal(v, wv)
    # lse: each exp and sum within a few float64 roundings of a positive sum of V terms (chains of 32 + 12), the logarithm one ulp
    live = ws > -np.inf
    assert np.array_equal(s == -np.inf, ~live)
    assert (np.abs(s[live] - ws[live]) <= 2.0 ** -53 * (100 + 8 * np.abs(ws[live]) + 8 * float(np.abs(x[np.isfinite(x)]).max()))).all()
    return s, b, v


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P,B,V,k", [(1, 1, 1, 1), (1, 1, 1, 5), (2, 3, 5, 7), (3, 2, 100, 4), (1, 4, 8191, 8), (2, 2, 8192, 32), (1, 5, 8193, 33),
                                     (2, 4, 50257, 8), (1, 8, 128256, 16), (1, 2, 32001, 64), (40, 3, 1001, 6), (1, 64, 500, 64), (300, 4, 64, 8)])
def test_beam_select(dev, P, B, V, k, dtype):
    rng = np.random.default_rng(V + k)
    x = rng.standard_normal((P, B, V)) * 3
    cum = -30 * rng.random((P, B))
    check_select(x, cum, k, dev, dtype)


@pytest.mark.parametrize("k", [1, 8, 40, 64])
def test_beam_select_ties_and_orders(dev, k):
    """Equal logits and beams, rising and falling rows, the best all in one thread's share, zeros of both signs."""
    V, B = 20000, 3
    i = np.arange(V)
    rows = [np.zeros(V), np.where(i % 2 == 0, 0.0, -0.0), i / V, -i / V, np.where(i % 1024 < 4, 5.0 + i / V, 0.0), np.where(i % 1024 == 7, i, -1.0),
            np.where(i // 4 % 256 == 3, 3.0, 3.0 - 1e-3), np.round(np.random.default_rng(0).standard_normal(V)), np.full(V, -3e38), np.where(i == V - 1, 3e38, -3e38)]
    for r in range(len(rows)):
        x = np.stack([rows[r], rows[(r + 1) % len(rows)], rows[r]])[None]
        check_select(x, np.array([[-1.0, -2.0, -1.0]]), k, dev)
        check_select(np.stack([rows[r]] * B)[None], np.zeros((1, B)), k, dev)      # beams alike: the first


def test_beam_select_without_enough(dev):
    """Rows with NaN, infinities or nothing, dead beams, fewer continuations than asked for."""
    V = 9000
    rng = np.random.default_rng(1)
    x = rng.standard_normal((7, 4, V))
    x[0, 1, 8500] = np.nan
    x[0, 2, 3] = np.inf
    x[0, 3] = -np.inf
    x[1, :, 5:] = -np.inf
    x[2] = -np.inf
    x[3, 0] = np.nan
    x[4, 1, 100:] = -np.inf
    cum = -rng.random((7, 4))
    cum[3, 1:] = -np.inf
    cum[4, [0, 2]] = -np.inf, np.nan
    cum[5, 1:] = -np.inf
    for k in (1, 8, 30):
        check_select(x, cum, k, dev)


def test_beam_scores_do_not_depend_on_the_batch(dev):
    g = torch.Generator(device=dev)
    g.manual_seed(4)
    x = 3 * torch.randn(300, 2, 40000, generator=g, device=dev)
    cum = -torch.rand(300, 2, dtype=F64, device=dev, generator=g)
    whole = ops.beam_select(x, cum, 4)
    for p in (0, 7, 299):
        one = ops.beam_select(x[p:p + 1].contiguous(), cum[p:p + 1].contiguous(), 4)
        assert all(torch.equal(a[0], b[p]) for a, b in zip(one, whole))


def test_beam_select_replayed(dev):
    x, cum = torch.randn(2, 3, 30000, device=dev), torch.zeros(2, 3, dtype=F64, device=dev)
    ops.beam_select(x, cum, 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.beam_select(x, cum, 6)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, device=dev))
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ops.beam_select(x, cum, 6)))


def test_beam_select_refuses(dev):
    x, cum = torch.zeros(2, 3, 10, device=dev), torch.zeros(2, 3, dtype=F64, device=dev)
    for a, b, k, text in ((x, cum, 0, "k is"), (x, cum, 65, "k is"), (x.half(), cum, 1, "dtype"), (x, cum.float(), 1, "float64"),
                          (x, cum[:1], 1, "scores must"), (x[0], cum, 1, "dims"), (x.transpose(1, 2), cum, 1, "contiguous"),
                          (torch.zeros(1, 65, 10, device=dev), torch.zeros(1, 65, dtype=F64, device=dev), 64, "4096")):
        with pytest.raises(ValueError, match=text):
            ops.beam_select(a, b, k)
    assert [t.shape for t in ops.beam_select(x[:0], cum[:0], 3)] == [(0, 3)] * 3


# ---------------------------------------------------------------- the engine
def _models():
    from draftkv.llama import demo_llama
    from draftkv.model import demo_model
    return {"llama": lambda: demo_llama(n_layers=2), "tiny": demo_model}


PROMPTS = [[5, 9, 2, 7, 7, 3, 1, 4, 8, 6, 2, 2, 5, 1, 9, 3, 3, 7, 20, 11], [3, 1, 4, 1, 5]]


@pytest.mark.parametrize("name", ["llama", "tiny"])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_samples(dev, name, temperature):
    """Drafted and plain continuations agree where they must (greedy), each prompt's pages are held once, and a continuation
    alone is the one it is among others."""
    from draftkv import CompressionConfig, DraftKVEngine, FixedPolicy
    m = _models()[name]()
    n, new = 3, 40
    run = lambda gamma, **kw: DraftKVEngine(m, FixedPolicy(CompressionConfig(4, 0.5), gamma), seed=5).generate_samples(PROMPTS, n, new, temperature, **kw)
    plain, drafted = run(0), run(4)
    for p, prompt in enumerate(PROMPTS):
        assert len(plain[p]) == n
        for r in plain[p] + drafted[p]:
            assert r.tokens[: len(prompt)] == prompt and len(r.tokens) == len(prompt) + new
    if temperature == 0.0:
        for p in range(len(PROMPTS)):
            assert all(r.tokens == plain[p][0].tokens for r in plain[p] + drafted[p])
    else:
        assert any(plain[0][0].tokens != r.tokens for r in plain[0][1:])
    e = DraftKVEngine(m, FixedPolicy(CompressionConfig(4, 0.5), 0), seed=5)
    e.generate_samples(PROMPTS[:1], n, new, temperature)
    full = e.last_full
    full.pools[0].check_invariants()
    whole = (len(PROMPTS[0]) - 1) // 16
    assert (full.pages[:, :whole] == full.pages[0, :whole]).all() and full.groups.max_shared >= 16 * whole
    assert e.generate_samples([], 2, 5) == []
    assert [[r.tokens for r in x] for x in e.generate_samples(PROMPTS, 2, 0, temperature)] == [[p, p] for p in PROMPTS]
    assert [list(r.tokens) for r in e.generate_samples(PROMPTS[:1], 1, 8, 0.0)[0]] == [plain_tokens(m, PROMPTS[0], 8)]


@pytest.mark.parametrize("name", ["llama", "tiny"])
def test_samples_of_one_token_prompts(dev, name):
    from draftkv import CompressionConfig, DraftKVEngine, FixedPolicy
    m = _models()[name]()
    runs = [DraftKVEngine(m, FixedPolicy(CompressionConfig(8, 0.9), gamma)).generate_samples([[7], [3, 4]], 3, 24, 0.0) for gamma in (0, 5)]
    for p in range(2):
        assert all(r.tokens == runs[0][p][0].tokens for x in runs for r in x[p])


def plain_tokens(m, prompt, new):
    """Greedy decoding over a shared cache of one sequence, token by token."""
    from draftkv import SharedKVCache
    c = SharedKVCache(m.n_layers, m.n_kv_heads, m.d_head, 16, 20, batch=1, device="cuda", chunk_keys=2048)
    toks = list(prompt)
    lg = m.forward(toks, c, 0)[-1]
    for _ in range(new):
        toks.append(int(np.argmax(lg)))
        lg = m.forward(toks[-1:], c, len(toks) - 1)[-1]
    return toks


def plain_beams(m, prompt, B, new, eos, penalty):
    """Beam search by whole forwards over the ordinary full cache, in float64."""
    from draftkv import FullKVCache

    def logp(tokens):
        c = FullKVCache(m.n_layers, m.n_kv_heads, m.d_head, device="cuda")
        x = m.forward(tokens, c, 0)[-1].astype(np.float64)
        return x - x.max() - math.log(np.exp(x - x.max()).sum())

    beams, ended, gap = [(0.0, list(prompt))], [], math.inf
    for i in range(new):
        cand = sorted(((-(s + lp[v]), j, v) for j, (s, t) in enumerate(beams) for lp in [logp(t)] for v in range(len(lp))))
        vals = [c[0] for c in cand[: 2 * B + 1]]
        gap = min([gap] + [b - a for a, b in zip(vals, vals[1:])])
        nxt = []
        for rank, (s, j, v) in enumerate(cand[: 2 * B]):
            if len(nxt) == B:
                break
            t = beams[j][1] + [v]
            if v == eos:
                if rank < B:
                    ended.append((-s / (i + 1) ** penalty, t))
                continue
            nxt.append((-s, t))
        beams = nxt
        ended = sorted(ended, key=lambda h: -h[0])[:B]
        if not beams or len(ended) == B and beams[0][0] / (i + 1) ** penalty <= ended[-1][0]:
            return ended, gap
    ended += [(s / new ** penalty, t) for s, t in beams]
    return sorted(ended, key=lambda h: -h[0])[:B], gap


@pytest.mark.parametrize("B,new,eos,penalty", [(1, 12, None, 1.0), (4, 10, None, 1.0), (3, 12, 17, 0.7), (5, 8, 3, 2.0), (2, 1, None, 0.0)])
@pytest.mark.parametrize("name", ["llama", "tiny"])
def test_beams(dev, name, B, new, eos, penalty):
    from draftkv import DraftKVEngine
    m = _models()[name]()
    if eos is not None:     # a token that the beams do meet
        eos = DraftKVEngine(m).generate_beams(PROMPTS[:1], 1, 4)[0][0].tokens[-1]
    e = DraftKVEngine(m)
    got = e.generate_beams(PROMPTS, B, new, eos, penalty)
    e.last_full.pools[0].check_invariants()
    for p, prompt in enumerate(PROMPTS):
        want, gap = plain_beams(m, prompt, B, new, eos, penalty)
        # scores of the two differ by the attention's and the products' float32 roundings, 1e-4 and less; nearer choices are not compared
        assert len(got[p]) == len(want)
        for h, (s, t) in zip(got[p], want):
            assert h.tokens[: len(prompt)] == prompt
            assert h.score == pytest.approx(h.logprob / (len(h.tokens) - len(prompt)) ** penalty)
            if gap > 1e-3:
                assert h.tokens == t and h.score == pytest.approx(s, abs=2e-3)
    one = e.generate_beams(PROMPTS[:1], B, new, eos, penalty)      # alone as among others
    assert [h.tokens for h in one[0]] == [h.tokens for h in got[0]] and [h.score for h in one[0]] == [h.score for h in got[0]]


def test_beams_of_nothing(dev):
    from draftkv import DraftKVEngine
    m = _models()["llama"]()
    h = DraftKVEngine(m).generate_beams([[3]], 2, 0)
    assert h[0][0].tokens == [3] and h[0][0].score == 0.0
    assert len(DraftKVEngine(m).generate_beams([[3]], 32, 3)[0]) == 32     # (more beams than the first step's tokens would do)


def test_a_bf16_model_samples(dev):
    from draftkv import CompressionConfig, DraftKVEngine, FixedPolicy
    from draftkv.llama import LlamaLike
    cfg = dict(num_hidden_layers=2, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=256,
               vocab_size=512, rms_norm_eps=1e-5, rope_theta=10000.0)
    m = LlamaLike.random(cfg, seed=1, std=0.1)
    prompt = [[(7 * i) % 500 for i in range(200)]]
    runs = [DraftKVEngine(m, FixedPolicy(CompressionConfig(8, 0.5, scale_fp16=True), g)).generate_samples(prompt, 4, 30, 0.0) for g in (0, 3)]
    assert all(r.tokens == runs[0][0][0].tokens for x in runs for r in x[0])
