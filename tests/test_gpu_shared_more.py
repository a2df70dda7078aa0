"""Attention over shared pages, page copies and the engine's calls over them at sizes and histories where they could go wrong: against
definitions in 64 bits, and against forwards of whole sequences."""

import math

import numpy as np
import pytest
import torch

from draftkv import ops

pytestmark = pytest.mark.gpu

F32, F64, BF16, I32 = torch.float32, torch.float64, torch.bfloat16, torch.int32
U = 2.0 ** -24


@pytest.mark.parametrize("extra", [-1, 0, 3])
def test_paged_copies_of_more_pages_than_a_launch_takes(dev, extra):
    """2^24 pairs of a workgroup each are 2^32 work-items, which no launch takes."""
    pairs, others = (1 << 24) + extra, 97
    store = torch.arange((pairs + others) * 4, dtype=I32, device=dev).view(-1, 4)
    dst = torch.arange(pairs, dtype=I32, device=dev)
    src = pairs + dst % others
    want = store.clone()
    want[:pairs] = store[src.long()]
    assert ops.paged_copy(store, src, dst) is store
    assert torch.equal(store, want)


def i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_bf16_queries_of_prompts(dev, dtype):
    """Inside filling() too, bf16 queries are taken, and a row is the one that it is outside."""
    from draftkv import SharedKVCache
    g = torch.Generator(device=dev)
    g.manual_seed(6)
    n, H, D = 70, 2, 64
    c = SharedKVCache(1, H, D, 16, 30, dtype, batch=2, max_tokens=100, device=dev)
    q, k, v = (torch.randn(2, n, h, D, generator=g, device=dev).to(BF16) for h in (8, H, H))
    count = i32([n, 20])
    c.reserve([n, n])
    with c.filling():
        out = c.append_attend(0, q, k, v, i32([0, 0]), n, count)
    assert out.dtype == BF16
    assert torch.equal(out, c.attend(0, q, i32([0, 0]), n, count=count))
    for s, m in enumerate((n, 20)):
        for t in (0, 1, 19):
            for h in range(8):
                kk, vv = k[s, : t + 1, h // 4].to(F64), v[s, : t + 1, h // 4].to(F64)
                w = torch.softmax(kk @ q[s, t, h].to(F64) / math.sqrt(D), 0)
                want, size = w @ vv, w @ vv.abs()
                # a score, a sum of 64 products of at most top in float32: 68 u top; twice, and in the exponent; probabilities hold two bf16
                # parts, the output one
                top = float((kk.abs() @ q[s, t, h].to(F64).abs()).max()) / math.sqrt(D)
                e = (2 * 72 * top + 64) * U + 2.0 ** -16
                assert ((out[s, t, h].to(F64) - want).abs() <= e * size + 2.0 ** -8 * (want.abs() + e * size)).all(), (s, t, h)


# ---------------------------------------------------------------- attention whose result is known to the last bits
DEAD = -16384.0      # K of a key that no row sees: with a query of 1/2 and more its probability is 0 in every type


def cache_of(H, D, bs, dtype, prefix, unit, K, V, CK, CV, n, own):
    """A prompt of the rows CK, CV [ctx, H, D] and n continuations with the first own[s] of the rows K, V [n, most, H, D]."""
    from draftkv import SharedKVCache
    ctx = CK.shape[0]
    pages = -(-ctx // bs) + n * (-(-K.shape[1] // bs) + 2)
    c = SharedKVCache(1, H, D, bs, pages, dtype, batch=1, max_tokens=ctx + K.shape[1], device="cuda", prefix_keys=prefix, unit_keys=unit)
    c.store.fill_(math.nan)
    if ctx:
        c.reserve([ctx])
        c.append_layer(0, CK[None], CV[None], i32([0]))
        c.commit([ctx])
    c.fork([0] * n)
    c.reserve(own)
    c.append_layer(0, K, V, i32([ctx] * n), i32(own))
    c.commit(own)
    return c


def counted(dev, seed, D, H, G, bs, dtype, qdtype, prefix, unit, ctx, n, own, T):
    """Keys that count fully or not at all, values that are whole numbers: every sum is exact, and a row is the sum of the values that it
    sees over their number, but for the division (half a step, one of float32 at most) and the output's rounding. A key or a value from
    another row, page or head, one too many or too few, is another number."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    most = max(own)

    def rows(*shape):
        live = torch.rand(*shape, H, generator=g, device=dev) < 0.5
        live[..., 0, :] = True
        k = torch.zeros(*shape, H, D, device=dev)
        k[..., seed % D] = torch.where(live, 0.0, DEAD)
        v = torch.randint(-128, 129, (*shape, H, D), generator=g, device=dev).float()
        return live.to(F64), k.to(dtype), v.to(dtype)

    cl, ck, cv = rows(max(ctx, 1))
    cl, ck, cv = cl[:ctx], ck[:ctx], cv[:ctx]
    ol, ok, ov = rows(n, most)
    c = cache_of(H, D, bs, dtype, prefix, unit, ok, ov, ck, cv, n, own)
    q = (0.5 + torch.rand(n, T, H * G, D, generator=g, device=dev)).to(qdtype)
    start = [ctx + o - T for o in own]
    out = c.attend(0, q, i32(start), max(start) + T)
    assert c.groups.max_shared == (ctx // bs * bs if n > 1 else 0)
    step = U * 2 if qdtype == F32 else 2.0 ** -8 + 2 * U
    for s in range(n):
        live, v = torch.cat([cl, ol[s]]), torch.cat([cv, ov[s]]).to(F64)
        total, number = torch.cumsum(v * live[..., None], 0), torch.cumsum(live, 0)
        at = torch.arange(start[s], start[s] + T, device=dev)
        want = (total[at] / number[at][..., None]).repeat_interleave(G, 1)
        err = (out[s].to(F64) - want).abs()
        assert (err <= step * want.abs()).all(), (s, float((err / want.abs().clamp(min=1e-30)).max()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,G,prefix,unit,ctx,n,own,T", [
    # pieces of the shared keys of 128 and 256 runs of 16, offsets of 64 of which a wave holds: waves apart (one and two tiles)
    (128, 4, 2048, 128, 5008, 3, 40, 1), (64, 3, 4096, 64, 9024, 20, 17, 1), (128, 4, 4096, 128, 8192, 5, 20, 2),
    # and four tiles over one ring
    (128, 4, 2048, 128, 6016, 32, 33, 1), (64, 4, 4096, 64, 9024, 5, 21, 5), (96, 2, 4096, 128, 5008, 9, 30, 9),
    # units of a sequence's own
    (128, 4, 2048, 2048, 64, 2, 5001, 1), (64, 1, 1024, 4096, 32, 2, 9003, 7), (32, 2, 2048, 4096, 0, 1, 5007, 16),
    (128, 4, 2048, 2048, 96, 2, 5001, 20), (64, 8, 1024, 4096, 0, 2, 9003, 9), (96, 3, 65536, 65536, 4000, 2, 4500, 40)])
def test_pieces_of_many_runs(dev, D, G, prefix, unit, ctx, n, own, T, dtype):
    counted(dev, D + T, D, 2, G, 16, dtype, F32, prefix, unit, ctx, n, [own - 13 * s % 12 for s in range(n)], T)


@pytest.mark.parametrize("seed", range(40))
def test_any_shape(dev, seed):
    """Sizes at random: widths, heads, blocks, types, pieces, lengths."""
    rng = np.random.default_rng(seed)
    pick = lambda *x: x[int(rng.integers(len(x)))]
    D = pick(1, 8, 32, 40, 64, 80, 96, 112, 128, int(rng.integers(1, 129)))
    T, n = pick(1, 1, 2, 5, 17), int(rng.integers(1, 12))
    own = [int(rng.integers(T, T + pick(3, 50, 400))) for _ in range(n)]
    counted(dev, seed, D, int(rng.integers(1, 4)), pick(1, 2, 3, 4, 8, 16), pick(16, 16, 16, 32, 48, 1, 5, 128), pick(F32, BF16), pick(F32, BF16),
            32 * int(rng.integers(1, 40)), 32 * int(rng.integers(1, 40)), pick(0, 1, 31, 32, 33, 500, int(rng.integers(1, 3000))), n, own, T)


@pytest.mark.parametrize("where", ["shared", "own"])
@pytest.mark.parametrize("D,G,n", [(64, 4, 4), (128, 8, 12), (40, 4, 8), (96, 32, 3)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_queries_and_probabilities_hold_24_bits(dev, dtype, D, G, n, where):
    """One key of score 0 and value 0 and one of score s = q a / sqrt(D) in -2.5 .. -0.6, the others of probability 0: out is v w / (1 + w)
    with w = e^s, and hardly anything is summed. With u = 2^-24: q log2(e) / sqrt(D) is off by 2 u (the constant and the product), its three
    parts are all of it, their products with a bf16 key are exact, and their sum is off by 4 u at most (two additions, cut or rounded): 6 u of
    |s| log2(e) <= 3.6, so 15 u of w; the exponential 2 u; the probability's parts and their sum as much as the query's, 4 u; 1 + w, the
    division and the merge 2 u each. In all less than 40 u of |out|. A query or a probability in two parts is off by 2^-17 and more (128 u;
    of 64 drawn ones the worst by 107 to 240 u, the middle one by 13 to 46)."""
    g = torch.Generator(device=dev)
    g.manual_seed(D + G)
    H, ctx, own, at = 2, 96, 40, 10
    a = float(torch.tensor(-1.25 * math.sqrt(D)).to(BF16))
    v = torch.randn(H, D, generator=g, device=dev).to(dtype)

    def rows(*shape, here):
        k = torch.zeros(*shape, H, D, device=dev)
        k[..., 3] = DEAD
        x = torch.randn(*shape, H, D, generator=g, device=dev)
        if here:
            k[..., at:at + 2, :, 3] = torch.tensor([0.0, a], device=dev)[:, None]
            x[..., at, :, :] = 0.0
            x[..., at + 1, :, :] = v.float()
        return k.to(dtype), x.to(dtype)

    ck, cv = rows(ctx, here=where == "shared")
    ok, ov = rows(n, own, here=where == "own")
    c = cache_of(H, D, 16, dtype, 64, 64, ok, ov, ck, cv, n, [own] * n)
    q = 0.5 + 1.5 * torch.rand(n, 1, H * G, D, generator=g, device=dev)
    assert q.shape[0] * q.shape[2] >= 32
    out = c.attend(0, q, i32([ctx + own - 1] * n), ctx + own)
    w = torch.exp(q[..., 3].to(F64) * a / math.sqrt(D))
    want = (w / (1 + w))[..., None] * v.to(F64).repeat_interleave(G, 0)
    err = (out.to(F64) - want).abs() / (U * want.abs())
    assert err.max() <= 40, float(err.max())


def test_a_pool_that_shrank(dev):
    """compact() to the live pages, between an append and the attention that reads it, and again after more rows."""
    from draftkv import SharedKVCache
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    c = SharedKVCache(3, 2, 64, 16, 90, BF16, batch=2, max_tokens=400, device=dev, prefix_keys=64, unit_keys=64)
    k, v = (torch.randn(2, 150, 2, 64, generator=g, device=dev) for _ in range(2))
    c.reserve([150, 100])
    for L in range(3):
        c.append_layer(L, k, v, i32([0, 0]), i32([150, 100]))
    c.commit([150, 100])
    c.fork([1, 1, 1])
    c.truncate([100, 90, 100])
    c.reserve([5, 30, 5])
    for L in range(3):
        c.append_layer(L, k[[1, 0, 1], :30].contiguous(), v[[1, 0, 1], :30].contiguous(), i32([100, 90, 100]), i32([5, 30, 5]))
    c.commit([5, 30, 5])
    q = torch.randn(3, 1, 8, 64, generator=g, device=dev)
    start = i32([104, 119, 104])
    want = [c.attend(L, q, start, 120) for L in range(3)]
    for n in (None, c.blocks_in_use, 200, c.blocks_in_use + 1):
        c.compact(n)
        assert int(c.d_tables.max()) < c.store.shape[0] and c.pages.max() < c.blocks_in_use
        for L in range(3):
            assert torch.equal(c.attend(L, q, start, 120), want[L])
    c.compact(20)
    c.reserve([30, 0, 30])
    for L in range(3):
        c.append_layer(L, k[:1, 40:70].expand(3, -1, -1, -1).contiguous(), v[:1, 40:70].expand(3, -1, -1, -1).contiguous(), i32([105, 0, 105]), i32([30, 0, 30]))
    c.commit([30, 0, 30])
    out = c.attend(1, q, i32([134, 119, 134]), 135)
    assert torch.equal(out[0], c.attend(1, q, i32([134, 119, 134]), 300)[0]) and torch.equal(out[1], want[1][1])
    kk, vv, _ = c.read(1, 2)
    assert np.array_equal(kk[105:], k[0, 40:70].to(BF16).float().cpu().numpy()) and np.array_equal(vv[:100], v[1, :100].to(BF16).float().cpu().numpy())


# ---------------------------------------------------------------- the engine, with prompts of more keys than a piece's step
def models():
    from draftkv.llama import demo_llama
    from draftkv.model import demo_model
    return {"llama": lambda: demo_llama(n_layers=2), "tiny": demo_model}


def prompts(seed):
    """130 and 75 tokens: 128 and 64 rows of them are whole pages, and whole steps of the walk."""
    return [np.random.default_rng(seed).integers(0, 128, n).tolist() for n in (130, 75)]


def whole(m, tokens):
    """float64 log probabilities behind every token, by one forward over an ordinary cache."""
    from draftkv import FullKVCache
    x = m.forward(tokens, FullKVCache(m.n_layers, m.n_kv_heads, m.d_head, device="cuda"), 0).astype(np.float64)
    x = x - x.max(-1, keepdims=True)
    return x - np.log(np.exp(x).sum(-1, keepdims=True))


NEAR = 1e-3      # logits by other sums of the same float32 terms differ by 1e-4 and less (as in the tests of short prompts)


@pytest.mark.parametrize("name", ["llama", "tiny"])
@pytest.mark.parametrize("gamma", [0, 4])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_samples_of_long_prompts(dev, name, gamma, temperature):
    """Every token is the one that whole forwards choose: the best, or, without drafts, the one that the sequence's random number falls on."""
    from draftkv import CompressionConfig, DraftKVEngine, FixedPolicy
    m, n, new, T = models()[name](), 4, 40, temperature
    e = DraftKVEngine(m, FixedPolicy(CompressionConfig(4, 0.5), gamma), seed=5)
    P = prompts(3)
    got = e.generate_samples(P, n, new, T)
    full = e.last_full
    full.pools[0].check_invariants()
    assert full.groups._host[0] == [0, n, 2 * n] and full.groups._host[1] == [128] * n + [64] * n
    assert (full.pages[:n, :8] == full.pages[0, :8]).all() and (full.pages[n:, :4] == full.pages[n, :4]).all()
    for p, prompt in enumerate(P):
        for i, r in enumerate(got[p]):
            assert r.tokens[: len(prompt)] == prompt and len(r.tokens) == len(prompt) + new
            lp = whole(m, r.tokens[:-1])[len(prompt) - 1:]
            t = np.array(r.tokens[len(prompt):])
            if T == 0.0:
                assert r.tokens == got[p][0].tokens
                assert (lp[np.arange(new), t] >= lp.max(-1) - NEAR).all()
            elif gamma == 0:
                u = np.random.default_rng(5 + p * n + i).random(new)
                pr = np.exp(lp / T)
                cdf = np.cumsum(pr / pr.sum(-1, keepdims=True), -1)
                hi = cdf[np.arange(new), t]
                lo = np.where(t > 0, cdf[np.arange(new), np.maximum(t - 1, 0)], 0.0)
                assert (lo - NEAR <= u).all() and (u <= hi + NEAR).all(), (p, i)
    if T == 0.0:
        again = DraftKVEngine(m, FixedPolicy(CompressionConfig(4, 0.5), 4 - gamma), seed=5).generate_samples(P, n, new, T)
        assert [[r.tokens for r in x] for x in again] == [[r.tokens for r in x] for x in got]
    else:
        assert len({tuple(r.tokens) for r in got[0]}) > 1


# B, new tokens, the prompt whose fourth token ends a beam, length penalty
BEAMS = [(1, 12, None, 1.0), (4, 10, None, 1.0), (3, 12, 0, 0.7), (5, 8, {"llama": 1, "tiny": 0}, 2.0), (2, 40, None, 1.0), (2, 40, 0, 0.5),
         (3, 40, None, 0.0)]


@pytest.mark.parametrize("B,new,eos,penalty", BEAMS)
@pytest.mark.parametrize("name", ["llama", "tiny"])
def test_beams_of_long_prompts(dev, name, B, new, eos, penalty):
    """Every hypothesis's score against a whole forward of its tokens; and where choices lie apart (for every set but the last, one prompt
    at least: worked out beforehand) the hypotheses against a search by whole forwards. Beams come to share what they generated."""
    from draftkv import DraftKVEngine
    from test_gpu_shared import plain_beams
    m = models()[name]()
    P = prompts({"llama": 1, "tiny": 28}[name])
    if eos is not None:
        of = eos[name] if isinstance(eos, dict) else eos
        eos = DraftKVEngine(m).generate_beams([P[of]], 1, 4)[0][0].tokens[-1]
    e = DraftKVEngine(m)
    got = e.generate_beams(P, B, new, eos, penalty)
    full = e.last_full
    full.pools[0].check_invariants()
    if B > 1:
        first, shared = full.groups._host
        assert first == [0, B, 2 * B] and shared[0] >= 128 and shared[B] >= 64
        assert new < 40 or eos is not None or shared[0] >= 144
    compared = 0
    for p, prompt in enumerate(P):
        for h in got[p]:
            assert h.tokens[: len(prompt)] == prompt and (eos is None or eos not in h.tokens[len(prompt): -1])
            lp = whole(m, h.tokens[:-1])[len(prompt) - 1:]
            assert h.logprob == pytest.approx(float(lp[np.arange(lp.shape[0]), h.tokens[len(prompt):]].sum()), abs=2 * NEAR)
            assert h.score == pytest.approx(h.logprob / lp.shape[0] ** penalty)
        assert len({tuple(h.tokens) for h in got[p]}) == len(got[p]) and [h.score for h in got[p]] == sorted((h.score for h in got[p]), reverse=True)
        want, gap = plain_beams(m, prompt, B, new, eos, penalty)
        assert len(got[p]) == len(want)
        if gap > NEAR:
            compared += 1
            assert [h.tokens for h in got[p]] == [t for _, t in want]
    assert compared > 0 or (B, new) == (3, 40)


# ---------------------------------------------------------------- beam selection at its largest
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P,B,V,k", [(1, 2, 1048576, 64), (1, 3, 1048573, 7), (20000, 3, 9, 3), (65535, 1, 5, 6), (2, 64, 8200, 64), (9, 7, 262145, 33)])
def test_beam_select_at_its_bounds(dev, P, B, V, k, dtype):
    from test_gpu_shared import check_select
    rng = np.random.default_rng(V + k)
    x = (rng.standard_normal((P, B, V), dtype=np.float32) * 2)
    check_select(x, -5 * rng.random((P, B)), k, dev, dtype)


@pytest.mark.parametrize("k", [2, 16, 64])
def test_beam_select_of_long_rows_of_equal_logits(dev, k):
    """Every tile of a row overflows its lists: steps, one value, two values, the last tile alone above."""
    from test_gpu_shared import check_select
    V = 300001
    i = np.arange(V)
    rows = [np.zeros(V), np.where(i % 3 == 1, 2.0, 1.0), (i // 4096).astype(np.float64), -(i // 20000).astype(np.float64), np.where(i >= V - 70, 1.0, 0.0),
            np.where(i < 50, 1.0, 0.0)]
    for a in rows:
        check_select(np.stack([a, rows[1], a])[None], np.array([[0.0, -0.25, 0.0]]), k, dev)


@pytest.mark.parametrize("name", ["llama", "tiny"])
@pytest.mark.parametrize("gamma", [0, 5])
def test_a_shared_cache_in_place_of_the_ordinary_one(dev, name, gamma):
    """full_cache_factory may make it: drafted and plain decoding of unlike prompts are the same."""
    from draftkv import CompressionConfig, DraftKVEngine, FixedPolicy, SharedKVCache
    m = models()[name]()
    P = prompts(9)
    make = lambda: SharedKVCache(m.n_layers, m.n_kv_heads, m.d_head, 16, 40, m.kv_dtype, batch=2, max_tokens=300, device=m.device)
    e = DraftKVEngine(m, FixedPolicy(CompressionConfig(4, 0.5), gamma), full_cache_factory=make)
    want = e.generate_baseline_batch(P, 40)
    got = e.generate_batch(P, 40)
    assert [list(r.tokens) for r in got] == want
    for p, t in zip(P, want):
        lp = whole(m, t[:-1])[len(p) - 1:]
        assert (lp[np.arange(40), t[len(p):]] >= lp.max(-1) - NEAR).all()
