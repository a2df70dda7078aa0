"""The full cache in 8 bits: append, attention, read, the mirror's sync from it and the engine over it, against the
definition in 64 bits. Queries read their own block in bf16 and the blocks before it as e4m3 codes times 2^e."""

import math

import numpy as np
import pytest
import torch

F32, F64, BF16, F8 = torch.float32, torch.float64, torch.bfloat16, torch.float8_e4m3fn


# ---------------------------------------------------------------- the definition
def coded(rows):
    """[bs, D] bf16 rows of a block of one head: the values its codes stand for, float64."""
    x = rows.to(F64)
    fine = torch.isfinite(x)
    amax = float(x[fine].abs().max()) if fine.any() else 0.0
    e = 0
    if amax > 0:
        m, ex = math.frexp(amax)          # amax = m 2^ex, 1/2 <= m < 1; 448 = 7/8 2^9
        e = min(max(ex - 9 if m <= 0.875 else ex - 8, -126), 119)
    y = x * 2.0 ** -e
    mag = y.abs()
    ex = torch.floor(torch.log2(torch.where(fine & (mag > 0), mag, torch.ones_like(mag)))).clamp(min=-6)
    step = torch.exp2(ex - 3)
    q = (torch.round(y / step) * step).clamp(-448, 448) * 2.0 ** e
    return torch.where(fine, q, torch.full_like(q, math.nan))


def values(rows, bs):
    """[n, H, D] bf16 rows of a sequence: (what sealed blocks stand for, the rows), float64; the open block as rows."""
    out = rows.to(F64)
    for j in range(rows.shape[0] // bs):
        for h in range(rows.shape[1]):
            out[j * bs:(j + 1) * bs, h] = coded(rows[j * bs:(j + 1) * bs, h])
    return out


def attention(q, k, v, first, bs):
    """q [T, Hq, D] at positions first.. of a sequence with bf16 rows k, v [n, H, D], float64. Also max |score|."""
    T, Hq, D = q.shape
    H = k.shape[1]
    k8, v8, k16, v16 = values(k, bs), values(v, bs), k.to(F64), v.to(F64)
    out = torch.zeros(T, Hq, D, dtype=F64)
    top = 0.0
    for t in range(T):
        p = first + t
        lim = p // bs * bs
        kk = torch.cat([k8[:lim], k16[lim:p + 1]])
        vv = torch.cat([v8[:lim], v16[lim:p + 1]])
        for h in range(Hq):
            s = kk[:, h * H // Hq] @ q[t, h].to(F64) / math.sqrt(D)
            top = max(top, float(s.abs().max()))
            out[t, h] = torch.softmax(s, 0) @ vv[:, h * H // Hq]
    return out, top


def bound(dtype, n, D, top, vmax, out):
    """float32: sums of n products and scores of D of them in float32 (24 bits; a score's error is an exponent's).
    bf16: each probability rounded once to bf16 (half a step of it is 2^-8) before the sum, and the result once."""
    f32 = 2.0 ** -24 * (4 * math.sqrt(n) + 4 * math.sqrt(D) * (1 + top)) * vmax
    return f32 if dtype == F32 else f32 + 2.0 ** -8 * vmax + 2.0 ** -8 * out.abs()


# ---------------------------------------------------------------- a cache with random rows
def rows_of(g, b, n, H, D, dev):
    k = torch.randn(b, n, H, D, generator=g, device=dev) * torch.exp(0.5 * torch.randn(H, D, generator=g, device=dev))
    v = torch.randn(b, n, H, D, generator=g, device=dev) * torch.exp(torch.randn(b, n, H, 1, generator=g, device=dev))
    return k, v


def new_cache(H, D, bs, n, b=1, layers=1, tail_rows=None, dev="cuda"):
    from draftkv.paged import PagedKVCache
    nb = -(-max(n, 1) // bs)
    return PagedKVCache(layers, H, D, bs, nb * layers, F8, batch=b, max_tokens=nb * bs, device=dev, tail_rows=tail_rows)


def i32(a, dev="cuda"):
    return torch.tensor(a, dtype=torch.int32, device=dev)


def fill(c, k, v, upto, layer=0):
    """The first upto[s] rows of each sequence, in one append."""
    T = max(upto)
    if T:
        c.append_layer(layer, k[:, :T].contiguous(), v[:, :T].contiguous(), i32([0] * len(upto)), i32(upto))


# ---------------------------------------------------------------- append and read
@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("D,H,dtype", [(128, 2, F32), (64, 3, BF16), (8, 2, F32), (80, 1, BF16), (256, 1, F32), (33, 2, F32)])
def test_append_codes_full_blocks(dev, bs, D, H, dtype):
    """Any cut of the rows into appends leaves the same values: those of the definition, bit for bit."""
    g = torch.Generator(device=dev)
    g.manual_seed(bs + D)
    n = 3 * bs + 5
    k, v = (x.to(dtype) for x in rows_of(g, 2, n, H, D, dev))
    k[0, 3, 0, 1] = 1e30       # a block of very different magnitudes
    v[1, :bs] = 0              # a block of zeros
    for cuts in ([n], [1] * (bs + 3) + [2 * bs + 2], [bs - 1, 2, bs, n - 2 * bs - 1], [5, n - 5]):
        c = new_cache(H, D, bs, n, b=2)
        c.reserve([n, n])
        at = 0
        for T in cuts:
            c.append_layer(0, k[:, at:at + T].contiguous(), v[:, at:at + T].contiguous(), i32([at, at]))
            at += T
        gk, gv = c.read_rows(0, i32([0, 0]), i32([n, n]), n + 3)
        for got, x in ((gk, k), (gv, v)):
            assert not got[:, n:].any()
            for s in range(2):
                assert torch.equal(got[s, :n].double().cpu(), values(x[s].to(BF16).cpu(), bs)), (cuts, s)


@pytest.mark.gpu
@pytest.mark.parametrize("bs,tail,D", [(64, 96, 40), (16, 32, 64), (32, 112, 24)])
def test_long_appends_wrap_around_the_tail(dev, bs, tail, D):
    """An append of more rows than the tail holds, begun inside a block: its codes come from the rows that were there and
    the new ones, and the tail then holds the last rows, those of the block before the last one too."""
    g = torch.Generator(device=dev)
    g.manual_seed(bs)
    for s0 in (1, 5, bs - 1, bs, bs + 17, 2 * bs + 3):
        for T in range(tail - bs + 2, tail + 2 * bs + 40, 11):
            n = s0 + T
            k, v = rows_of(g, 1, n, 2, D, dev)
            c = new_cache(2, D, bs, n, tail_rows=tail)
            for lo, hi in ((0, s0), (s0, n)):
                c.reserve([hi - lo])
                c.append_layer(0, k[:, lo:hi].contiguous(), v[:, lo:hi].contiguous(), i32([lo]))
                c.commit([hi - lo])
            for cut in (n, n - 1, n - n % bs - 1):
                if cut < 1 or cut // bs * bs < -(-n // 16) * 16 - tail:
                    continue
                gk, gv = c.read_rows(0, i32([0]), i32([cut]), cut)
                for got, x in ((gk, k), (gv, v)):
                    assert torch.equal(got[0].double().cpu(), values(x[0, :cut].to(BF16).cpu(), bs)), (s0, T, cut)


@pytest.mark.gpu
def test_append_values_that_are_not_finite(dev):
    """NaN and infinities become NaN codes and do not count for the scale; the smallest and largest magnitudes hold."""
    bs, H, D = 16, 1, 32
    k = torch.randn(1, 32, H, D, device=dev)
    v = torch.randn(1, 32, H, D, device=dev)
    k[0, 3, 0, 7], k[0, 4, 0, 1], k[0, 5, 0, 2] = math.inf, -math.inf, math.nan
    v[0, :16] = torch.randn(16, H, D, device=dev) * 2.0 ** -130      # bf16 subnormals
    v[0, 16:] = 3.38e38
    c = new_cache(H, D, bs, 32)
    c.reserve([32])
    c.append_layer(0, k, v, i32([0]))
    gk, gv = c.read_rows(0, i32([0]), i32([32]), 32)
    for got, x in ((gk, k), (gv, v)):
        want = values(x[0].to(BF16).cpu(), bs)
        assert torch.equal(torch.nan_to_num(got[0].double().cpu(), nan=123.0), torch.nan_to_num(want, nan=123.0))


@pytest.mark.gpu
def test_read_is_the_batch_one_protocol_too(dev):
    from draftkv import FullKVCache
    c = FullKVCache(2, dtype=F8, device=dev)
    k = np.random.default_rng(0).standard_normal((37, 2, 16)).astype(np.float32)
    for L in range(2):
        c.append(L, k[:30] + L, k[:30], np.arange(30))
        c.append(L, k[30:] + L, k[30:], np.arange(30, 37))
    for L in range(2):
        gk, gv, pos = c.read(L)
        assert pos.tolist() == list(range(37))
        assert np.array_equal(gk, values(torch.from_numpy(k + L).to(BF16), 16).numpy().astype(np.float32))
        assert np.array_equal(gv, values(torch.from_numpy(k).to(BF16), 16).numpy().astype(np.float32))


# ---------------------------------------------------------------- attention
# D, KV heads, query heads per KV head, block, rows per sequence that are there, new rows
SHAPES = [
    (128, 2, 4, 16, [0, 1, 15, 40], 1), (128, 2, 4, 16, [2047, 2048, 2049, 300], 5), (128, 1, 4, 16, [4100, 17, 0, 255], 17),
    (64, 3, 3, 32, [100, 31, 32, 600], 1), (64, 1, 1, 16, [0, 5, 16, 260], 16), (64, 2, 8, 128, [129, 127, 400, 0], 40),
    (8, 2, 4, 16, [33, 0, 7, 90], 3), (16, 4, 1, 16, [50, 49, 48, 47], 2), (256, 1, 2, 64, [300, 64, 63, 1], 9),
    (192, 2, 3, 16, [20, 40, 2060, 0], 4), (80, 1, 5, 32, [95, 96, 97, 3], 33), (33, 1, 2, 16, [70, 16, 0, 31], 1),
    (128, 2, 4, 64, [0, 0, 0, 0], 300), (64, 1, 12, 16, [700, 0, 33, 2000], 150),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"d{s[0]}h{s[1]}x{s[2]}b{s[3]}t{s[5]}")
def test_attention_against_64_bits(dev, shape, dtype):
    D, H, G, bs, have, T = shape
    b = len(have)
    g = torch.Generator(device=dev)
    g.manual_seed(D * 1000 + T)
    n = max(have) + T
    k, v = rows_of(g, b, n, H, D, dev)
    q = torch.randn(b, T, H * G, D, generator=g, device=dev).to(dtype)
    c = new_cache(H, D, bs, n, b=b)
    c.reserve([n] * b)
    fill(c, k, v, have)
    kn = torch.stack([k[s, have[s]:have[s] + T] for s in range(b)])
    vn = torch.stack([v[s, have[s]:have[s] + T] for s in range(b)])
    out = c.append_attend(0, q, kn, vn, i32(have), n)
    assert out.dtype == dtype
    for s in range(b):
        m = have[s] + T
        steps = list(range(T)) if T <= 40 else [0, 1, 15, 16, 63, 64, 65, T // 2, T - 2, T - 1]
        for t in steps:
            kk, vv = k[s, :m].to(BF16).cpu(), v[s, :m].to(BF16).cpu()
            want, top = attention(q[s, t:t + 1].cpu(), kk, vv, have[s] + t, bs) if D <= 64 or t in (0, T - 1) or T <= 5 else (None, 0)
            if want is None:
                continue
            err = (out[s, t].double().cpu() - want[0]).abs()
            tol = bound(dtype, have[s] + t + 1, D, top, float(vv.float().abs().max()), want[0])
            assert (err <= tol).all(), (s, t, float(err.max()), float(tol.max() if torch.is_tensor(tol) else tol))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(64, 1, 4, 16, 700, 1), (128, 1, 4, 16, 2500, 5), (128, 2, 4, 64, 300, 40), (256, 1, 2, 32, 400, 3),
                                   (192, 1, 1, 16, 2100, 9), (24, 1, 3, 128, 900, 30)], ids=lambda s: f"d{s[0]}n{s[4]}t{s[5]}")
def test_bf16_queries_are_off_by_the_outputs_rounding(dev, shape):
    """The probabilities of bf16 queries hold 16 bits: half a step of the bf16 output (2^-8 of it) is all that may show.
    Scores near each other, so that many keys take part and their values cancel."""
    D, H, G, bs, have, T = shape
    g = torch.Generator(device=dev)
    g.manual_seed(D + have)
    n = have + T
    k, v = (torch.randn(1, n, H, D, generator=g, device=dev) for _ in range(2))
    q = (0.2 * torch.randn(1, T, H * G, D, generator=g, device=dev)).to(BF16)
    c = new_cache(H, D, bs, n)
    c.reserve([n])
    fill(c, k, v, [have])
    out = c.append_attend(0, q, k[:, have:].contiguous(), v[:, have:].contiguous(), i32([have]), n)[0].double().cpu()
    k16, v16 = k[0].to(BF16).cpu(), v[0].to(BF16).cpu()
    want, top = attention(q[0].cpu(), k16, v16, have, bs)
    size, _ = attention(q[0].cpu(), k16, v16.abs(), have, bs)       # sum of p |v|
    # two bf16 parts of a probability leave 2^-8 of 2^-8 of it; float32 sums and scores as in bound()
    assert ((out - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * size + bound(F32, n, D, top, size, None)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,H,G,bs,n", [(128, 2, 4, 16, 2300), (64, 3, 3, 64, 700), (8, 1, 4, 16, 100), (256, 1, 1, 128, 520)])
def test_rows_do_not_depend_on_the_call(dev, D, H, G, bs, n, dtype):
    """Bit for bit the same rows from one call, from calls of a few, from one-row calls, and after appending other rows
    and rolling them back."""
    g = torch.Generator(device=dev)
    g.manual_seed(n)
    k, v = rows_of(g, 1, n, H, D, dev)
    junk = 100 * torch.randn(1, 40, H, D, generator=g, device=dev)
    q = torch.randn(1, n, H * G, D, generator=g, device=dev).to(dtype)
    whole = new_cache(H, D, bs, n + 64)
    whole.reserve([n + 64])
    ref = whole.append_attend(0, q, k, v, i32([0]), n)
    c = new_cache(H, D, bs, n + 64)
    c.reserve([n + 64])
    at, step = max(n - 150, 40), 0
    fill(c, k, v, [at])
    while at < n:
        c.append_layer(0, junk[:, :30].contiguous(), junk[:, :30].contiguous(), i32([at]))     # rejected rows
        T = min([1, 5, 1, 2, 17, 9][step % 6], n - at)
        out = c.append_attend(0, q[:, at:at + T].contiguous(), k[:, at:at + T].contiguous(), v[:, at:at + T].contiguous(),
                              i32([at]), n + 64 if step % 2 else at + T)
        assert torch.equal(out, ref[:, at:at + T]), (at, T)
        at, step = at + T, step + 1


# D, KV heads, query heads per KV head, block, rows that are there, new rows: prompts enough to fill the chip, and long ones
# of few sequences, whose keys several workgroups share
PROMPTS = [
    (128, 2, 8, 16, [0, 7, 30, 16, 100, 33], 300), (64, 2, 16, 32, [0, 7, 30, 16, 3, 2, 1, 31], 200), (16, 4, 16, 16, [20, 7, 1, 16, 3, 2, 0, 0], 300),
    (192, 2, 8, 64, [0, 7, 70, 64, 3, 2, 1, 129], 300), (256, 2, 8, 16, [0, 7, 30, 16, 3, 15], 200), (16, 4, 16, 16, [1700, 0, 2000, 1999], 200),
    (64, 2, 16, 16, [1700, 0, 3000, 2049], 200), (64, 1, 16, 128, [1700, 0, 3000, 2049], 200), (128, 2, 16, 16, [1700, 0, 2000, 1999], 200),
    (128, 1, 16, 64, [3000], 800), (192, 1, 16, 16, [2000], 800), (256, 1, 16, 16, [3000], 400), (256, 1, 8, 32, [3001], 800),
    (128, 1, 16, 16, [3000], 1200), (192, 1, 1, 16, [3000, 2990], 4000), (256, 1, 1, 64, [3000, 2990], 4000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", PROMPTS, ids=lambda s: f"d{s[0]}h{s[1]}x{s[2]}b{s[3]}t{s[5]}n{s[4][-1]}")
def test_prompts_equal_calls_of_a_few_rows(dev, shape, dtype):
    """Bit for bit, in every sequence, with values that are not finite in two of them; the last one's rows end early."""
    D, H, G, bs, have, T = shape
    b, m = len(have), max(have) + T
    g = torch.Generator(device=dev)
    g.manual_seed(D + T + b)
    k, v = rows_of(g, b, m, H, D, dev)
    for s, bad in ((0, have[0] + T // 2), (b // 2, have[b // 2] + T // 3)):
        k[s, bad, 0, 3], v[s, bad + 20, H - 1, 5] = math.nan, math.inf
    q = torch.randn(b, T, H * G, D, generator=g, device=dev).to(dtype)
    cnt = [T] * (b - 1) + [T - 21]

    def call(at, rows, count):
        """Rows at[s] .. of the sequences in one call, over a cache that holds those before them."""
        c = new_cache(H, D, bs, m, b=b)
        c.reserve([m] * b)
        fill(c, k, v, at)
        pick = lambda x: torch.stack([torch.nn.functional.pad(x[s, at[s]:at[s] + rows], (0, 0, 0, 0, 0, rows - x[s, at[s]:at[s] + rows].shape[0]))
                                      for s in range(b)])
        off = [a - h for a, h in zip(at, have)]
        qq = torch.stack([q[s, off[s]:off[s] + rows] for s in range(b)])
        return c.append_attend(0, qq, pick(k), pick(v), i32(at), max(at) + rows, i32(count))

    out = call(have, T, cnt)
    for t in (0, 1, T // 3 - 1, T // 2 - 2, T // 2 + 18, 130, T - 23 - 3):
        few = call([h + t for h in have], 3, [3] * b)
        got = out[:, t:t + 3]
        assert torch.equal(got.isnan(), few.isnan()) and torch.equal(got.nan_to_num(nan=0.0), few.nan_to_num(nan=0.0)), t


@pytest.mark.gpu
def test_a_bound_that_is_too_short_drops_chunks_only(dev):
    """max_len below what a sequence holds: its rows see the chunks of 2048 keys up to it and their own block."""
    D, H, G, bs, n = 64, 2, 2, 16, 5000
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    k, v = rows_of(g, 1, n + 1, H, D, dev)
    q = torch.randn(1, 1, H * G, D, generator=g, device=dev)
    c = new_cache(H, D, bs, n + 1)
    c.reserve([n + 1])
    fill(c, k, v, [n])
    out = c.append_attend(0, q, k[:, n:].contiguous(), v[:, n:].contiguous(), i32([n]), 100)
    own = n // bs * bs
    kk = torch.cat([k[0, :2048], k[0, own:n + 1]]).to(BF16).cpu()
    vv = torch.cat([v[0, :2048], v[0, own:n + 1]]).to(BF16).cpu()
    want, top = attention(q[0].cpu(), kk, vv, kk.shape[0] - 1, bs)
    assert ((out[0].double().cpu() - want).abs() <= bound(F32, kk.shape[0], D, top, float(vv.float().abs().max()), want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 40, 200])
def test_padding_rows_and_empty_sequences(dev, T):
    """Rows past count see what the last row does, a sequence without new rows gives zeros; no other block is touched."""
    D, H, G, bs = 64, 2, 2, 16
    g = torch.Generator(device=dev)
    g.manual_seed(T)
    have, cnt = [0, 100, 0, 33], [T, 1, 0, 0]
    n = 100 + T
    k, v = rows_of(g, 4, n, H, D, dev)
    q = torch.randn(4, T, H * G, D, generator=g, device=dev)
    q[:, 1:] = q[:, :1]        # the same query in every row: a padding row is then the last row again
    c = new_cache(H, D, bs, n, b=4)
    c.reserve([n] * 4)
    fill(c, k, v, have)
    kn = torch.stack([k[s, have[s]:have[s] + T] for s in range(4)])
    vn = torch.stack([v[s, have[s]:have[s] + T] for s in range(4)])
    kn[1, 1:], vn[1, 1:], kn[2], vn[2], kn[3] = math.nan, math.nan, math.nan, math.inf, math.nan
    before = c.store.clone()
    out = c.append_attend(0, q, kn, vn, i32(have), n, i32(cnt))
    assert torch.isfinite(out).all()
    assert not out[2:].any()
    for s, m in ((1, 101),):
        want, top = attention(q[s, :1].cpu(), k[s, :m].to(BF16).cpu(), v[s, :m].to(BF16).cpu(), m - 1, bs)
        err = (out[s].double().cpu() - want).abs().max()
        assert err <= bound(F32, m, D, top, float(v[s].abs().max()), want)
        assert torch.equal(out[s], out[s, :1].expand_as(out[s]))
    per = c.n_blocks
    assert torch.equal(c.store[2 * per:], before[2 * per:])      # no block of sequences 2 and 3 filled up


@pytest.mark.gpu
@pytest.mark.parametrize("D,T,have", [(128, 6, 30), (64, 40, 100), (128, 90, 10)])
def test_not_finite_values_stay_with_the_rows_that_see_them(dev, D, T, have):
    """NaN or infinity in K or V of a position: rows before it are as without, rows from it on are NaN (or hold the
    infinity's channel)."""
    H, G, bs = 1, 4, 16
    g = torch.Generator(device=dev)
    g.manual_seed(T)
    n = have + T
    k, v = rows_of(g, 1, n, H, D, dev)
    q = torch.randn(1, T, G, D, generator=g, device=dev)
    outs = []
    bad = have + T // 2
    for what in ("none", "v_nan", "v_inf", "k_nan"):
        kk, vv = k.clone(), v.clone()
        if what[0] == "v":
            vv[0, bad, 0, 5] = math.nan if what == "v_nan" else math.inf
        elif what == "k_nan":
            kk[0, bad, 0, 3] = math.nan
        c = new_cache(H, D, bs, n)
        c.reserve([n])
        fill(c, kk, vv, [have])
        outs.append(c.append_attend(0, q, kk[:, have:].contiguous(), vv[:, have:].contiguous(), i32([have]), n))
    clean, vnan, vinf, knan = outs
    m = bad - have
    for o in outs[1:]:
        assert torch.equal(o[:, :m], clean[:, :m])
    assert vnan[0, m:, :, 5].isnan().all() and knan[0, m:].isnan().all()
    others = [d for d in range(D) if d != 5]
    assert torch.isfinite(vnan[0, m:][:, :, others]).all()
    same_block = slice(m, min(T, (bad // bs + 1) * bs - have))
    assert torch.isinf(vinf[0, same_block, :, 5]).all()          # coded, an infinity is NaN


@pytest.mark.gpu
def test_rows_outside_the_block_table_are_none(dev):
    c = new_cache(1, 32, 16, 64, b=3)
    c.reserve([64] * 3)
    x = torch.randn(3, 20, 1, 32, device=dev)
    before = c.store.clone(), c.tail.clone()
    out = c.append_attend(0, x, x, x, i32([-1, 45, 1 << 30]), 64)
    assert not out.any() and torch.equal(c.store, before[0]) and torch.equal(c.tail, before[1])
    assert not c.read_rows(0, i32([-5, 64, 1 << 30]), i32([0, 100, (1 << 31) - 1]), 4)[0].any()


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """A sequence whose blocks lie past 4 GiB of the pool."""
    from draftkv.paged import PagedKVCache
    H, D, bs, n = 8, 128, 16, 200
    per = int(33000 * 33) // 8
    c = PagedKVCache(1, H, D, bs, per, F8, batch=1, max_tokens=bs * 32, device=dev)
    assert c.store.numel() > 1 << 32
    c.reserve([bs * 32])                     # the highest blocks first
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    k, v = rows_of(g, 1, n, H, D, dev)
    q = torch.randn(1, n, H, D, generator=g, device=dev)
    out = c.append_attend(0, q, k, v, i32([0]), n)
    small = new_cache(H, D, bs, n)
    small.reserve([n])
    assert torch.equal(out, small.append_attend(0, q, k, v, i32([0]), n))


@pytest.mark.gpu
def test_layers_and_sequences_do_not_mix(dev):
    D, H, G, bs, n, L = 64, 2, 2, 32, 150, 3
    g = torch.Generator(device=dev)
    g.manual_seed(9)
    many = new_cache(H, D, bs, n, b=3, layers=L)
    many.reserve([n] * 3)
    ins, outs = [], []
    for layer in range(L):
        k, v = rows_of(g, 3, n, H, D, dev)
        q = torch.randn(3, n, H * G, D, generator=g, device=dev)
        ins.append((q, k, v))
        outs.append(many.append_attend(layer, q, k, v, i32([0] * 3), n))
    for layer in range(L):
        q, k, v = ins[layer]
        for s in range(3):
            one = new_cache(H, D, bs, n)
            one.reserve([n])
            ref = one.append_attend(0, q[s:s + 1].contiguous(), k[s:s + 1].contiguous(), v[s:s + 1].contiguous(), i32([0]), n)
            assert torch.equal(outs[layer][s], ref[0])
            gk, gv = many.read_rows(layer, i32([0] * 3), i32([n] * 3), n)
            assert torch.equal(gk[s].double().cpu(), values(k[s].to(BF16).cpu(), bs))
    many.commit([n] * 3)
    rk, _, _ = many.read(1, seq=2)
    assert np.array_equal(rk, values(ins[1][1][2].to(BF16).cpu(), bs).float().numpy())


@pytest.mark.gpu
def test_another_stream_and_graph_replays(dev):
    """One-row steps recorded once and replayed at moving positions, with other work between, equal eager steps."""
    from draftkv import ops
    D, H, G, bs, n0, steps = 64, 2, 4, 16, 300, 40
    g = torch.Generator(device=dev)
    g.manual_seed(4)
    k, v = rows_of(g, 2, n0 + steps, H, D, dev)
    q = torch.randn(2, steps, H * G, D, generator=g, device=dev)
    N = n0 + steps
    caches = [new_cache(H, D, bs, N, b=2) for _ in range(2)]
    for c in caches:
        c.reserve([N, N])
        fill(c, k, v, [n0, n0])
    eager = [caches[0].append_attend(0, q[:, t:t + 1].contiguous(), k[:, n0 + t:n0 + t + 1].contiguous(),
                                     v[:, n0 + t:n0 + t + 1].contiguous(), i32([n0 + t] * 2), N) for t in range(steps)]
    qb, kb, vb, st = (torch.zeros_like(x) for x in (q[:, :1], k[:, :1], v[:, :1], i32([0, 0])))
    graph, ws = torch.cuda.CUDAGraph(), ops.Workspace()
    st.fill_(n0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), ops.private_workspace(ws):
        caches[1].append_attend(0, qb, kb, vb, st, N)
    torch.cuda.current_stream().wait_stream(side)
    with ops.private_workspace(ws), torch.cuda.graph(graph):
        out = caches[1].append_attend(0, qb, kb, vb, st, N)
    for t in range(steps):
        qb.copy_(q[:, t:t + 1])
        kb.copy_(k[:, n0 + t:n0 + t + 1])
        vb.copy_(v[:, n0 + t:n0 + t + 1])
        st.fill_(n0 + t)
        graph.replay()
        assert torch.equal(out, eager[t]), t


# ---------------------------------------------------------------- cache, mirror, engine
@pytest.mark.gpu
def test_long_rows_of_another_append_are_refused(dev):
    """The bf16 rows of a long append are there until the next one; short ones are in the tail."""
    T = 150
    c = new_cache(1, 32, 16, 400, layers=2)
    k = torch.randn(1, T, 1, 32, device=dev)
    c.reserve([T + 2])
    st = i32([0])
    with pytest.raises(ValueError, match="append_layer"):
        c.attend(0, k, st, T)
    # each within bound() of the same exact result, which -v negates; |score| <= |k|^2 / sqrt(D)
    tol = 2 * bound(F32, T, 32, float(k.norm(dim=-1).max()) ** 2 / math.sqrt(32), float(k.abs().max()), None)
    c.append_layer(0, k, k, st)
    a = c.attend(0, k, st, T)
    c.append_layer(1, k, -k, st)
    with pytest.raises(ValueError, match="append_layer"):
        c.attend(0, k, st, T)
    b = c.attend(1, k, st, T)
    one = new_cache(1, 32, 16, 400)       # (a matrix instruction need not round -x as it rounds x)
    one.reserve([T])
    assert torch.equal(b, one.append_attend(0, k, k, -k, st, T)) and ((a + b).abs() <= tol).all()
    with pytest.raises(ValueError, match="queries"):
        c.append_attend(0, k[:, :3].contiguous(), k, k, st, T)
    for L in range(2):     # short ones: any order
        c.append_layer(L, k[:, :2].contiguous(), (1 - 2 * L) * k[:, :2], i32([T]))
    x, y = (c.attend(L, k[:, :2].contiguous(), i32([T]), T + 2) for L in range(2))
    assert ((x + y).abs() <= tol).all()


@pytest.mark.gpu
def test_long_rows_from_another_start_are_refused(dev):
    """attend() of a long append's rows: the same layer, T, start and count, and nothing on that layer in between."""
    T, D = 150, 32
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    k, v = rows_of(g, 1, 3 * T, 1, D, dev)
    q = torch.randn(1, T, 2, D, generator=g, device=dev)
    part = lambda x, i: x[:, T * i:T * i + T].contiguous()
    c, ref = (new_cache(1, D, 16, 4 * T) for _ in range(2))
    for x in (c, ref):
        x.reserve([3 * T])
    st = [i32([0]), i32([T])]
    for i in range(2):
        c.append_layer(0, part(k, i), part(v, i), st[i])
        want = ref.append_attend(0, q, part(k, i), part(v, i), st[i], 2 * T)
    with pytest.raises(ValueError, match="append_layer"):
        c.attend(0, q, st[0], 2 * T)
    with pytest.raises(ValueError, match="append_layer"):
        c.attend(0, q, st[1], 2 * T, count=i32([T - 1]))
    for start, count in ((st[1], None), (st[1].clone(), None), (st[1], i32([T]))):
        assert torch.equal(c.attend(0, q, start, 2 * T, count=count), want)
    with pytest.raises(ValueError, match="must match"):
        c.append_layer(0, part(k, 1), part(v, 1)[..., :8].contiguous(), st[1])
    with pytest.raises(ValueError, match="append_layer"):
        c.attend(0, q, st[1], 2 * T)
    c.append_layer(0, part(k, 1), part(v, 1), st[1])
    st[1].add_(1)
    for start in (st[1], i32([T]), i32([T + 1])):
        with pytest.raises(ValueError, match="append_layer"):
            c.attend(0, q, start, 2 * T)
    with torch.inference_mode():
        a, b = i32([T]), i32([T])
        c.append_layer(0, part(k, 1), part(v, 1), a)
        assert torch.equal(c.attend(0, q, b, 2 * T), want)
    for change in (lambda: c.append_layer(0, part(k, 2)[:, :1].contiguous(), part(v, 2)[:, :1].contiguous(), i32([T])),
                   lambda: (c.commit([T + 3]), c.truncate([T]))):
        s = i32([T])
        c.append_layer(0, part(k, 1), part(v, 1), s)
        change()
        with pytest.raises(ValueError, match="append_layer"):
            c.attend(0, q, s, 2 * T)


@pytest.mark.gpu
def test_a_replayed_long_append_leaves_the_eager_rows(dev):
    """A graph's long append to one layer, replayed between an eager one to another layer and its attend()."""
    T, D = 150, 32
    g = torch.Generator(device=dev)
    g.manual_seed(8)
    k, v = rows_of(g, 1, 2 * T, 1, D, dev)
    q = torch.randn(1, T, 2, D, generator=g, device=dev)
    a, b = (tuple(x[:, lo:lo + T].contiguous() for x in (k, v)) for lo in (0, T))
    c, ref = (new_cache(1, D, 16, 2 * T, layers=2) for _ in range(2))
    for x in (c, ref):
        x.reserve([T])
    st = i32([0])
    c.append_attend(0, q, *a, st, T)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.append_layer(0, *a, st)
        out = c.attend(0, q, st[:], T)      # (a view of it)
        with pytest.raises(ValueError, match="append_layer"):
            c.attend(1, q, st, T)
    want = [ref.append_attend(0, q, *a, st, T), ref.append_attend(1, q, *b, st, T)]
    for _ in range(3):
        c.append_layer(1, *b, st)
        graph.replay()
        assert torch.equal(c.attend(1, q, st, T), want[1])
        assert torch.equal(out, want[0])


@pytest.mark.gpu
def test_a_captured_long_append_keeps_its_rows(dev):
    """A longer append after the capture moves the bf16 rows; the graph still has its own."""
    T, D = 150, 32
    g = torch.Generator(device=dev)
    g.manual_seed(9)
    k, v = rows_of(g, 1, 700, 2, D, dev)
    q = torch.randn(1, T, 4, D, generator=g, device=dev)
    c, other = (new_cache(2, D, 16, 1000) for _ in range(2))
    for x in (c, other):
        x.reserve([700])
    kb, vb, st = k[:, :T].clone(), v[:, :T].clone(), i32([0])
    want = c.append_attend(0, q, kb, vb, st, T)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.append_attend(0, q, kb, vb, st, T)
    c.append_layer(0, k, v, st)                                     # moves them
    junk = [torch.full((1 << 20,), math.nan, device=dev) for _ in range(8)]   # takes what was freed
    for i in range(3):
        kb.copy_(k[:, T * i:T * i + T])
        vb.copy_(v[:, T * i:T * i + T])
        want = other.append_attend(0, q, kb, vb, st, T)
        graph.replay()
        assert torch.equal(out, want)
    assert all(x.isnan().all() for x in junk)


@pytest.mark.gpu
def test_truncate_keeps_what_the_tail_holds(dev):
    c = new_cache(2, 16, 16, 400, tail_rows=64)
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    k, v = rows_of(g, 1, 400, 2, 16, dev)
    for lo, hi in ((0, 250), (250, 253)):
        c.reserve([hi - lo])
        c.append_layer(0, k[:, lo:hi].contiguous(), v[:, lo:hi].contiguous(), i32([lo]))
        c.commit([hi - lo])
    with pytest.raises(ValueError, match="bf16 rows of that block are gone"):
        c.truncate(180)                    # 256 - 64 = 192 on
    assert c.length == 253
    for cut in (200, 193, 96):             # inside a held block, and to a block's end
        c.truncate(cut)
        gk, _, _ = c.read(0)
        assert np.array_equal(gk, values(k[0, :cut].to(BF16).cpu(), 16).float().numpy())
    with pytest.raises(ValueError, match="gone"):
        c.truncate(90)
    c.reserve([300])
    q = torch.randn(1, 300, 4, 16, generator=g, device=dev)
    out = c.append_attend(0, q, k[:, 96:396].contiguous(), v[:, 96:396].contiguous(), i32([96]), 396)
    ref = new_cache(2, 16, 16, 400)
    ref.reserve([396])
    fill(ref, k, v, [96])
    assert torch.equal(out, ref.append_attend(0, q, k[:, 96:396].contiguous(), v[:, 96:396].contiguous(), i32([96]), 396))


@pytest.mark.gpu
@pytest.mark.parametrize("bits,keep,D", [(4, 0.5, 64), (8, 1.0, 128), (16, 0.25, 16)])
def test_mirror_from_it_equals_the_mirror_from_its_values(dev, bits, keep, D):
    """sync_from and rebuild_layers over the 8-bit cache give the mirror that a float32 cache holding the same values
    gives, codes and scores alike."""
    from draftkv import CompressedKVCache, CompressionConfig, PagedKVCache
    H, L, b, n, bs = 2, 2, 2, 150, 16
    g = torch.Generator(device=dev)
    g.manual_seed(bits)
    c = new_cache(H, D, bs, 200, b=b, layers=L)
    f = PagedKVCache(L, H, D, bs, L * 13, torch.float32, batch=b, max_tokens=208, device=dev)

    def grow(lo, hi):
        for x in (c, f):
            x.reserve([hi - lo] * b)
        for layer in range(L):
            k, v = rows_of(g, b, hi - lo, H, D, dev)
            c.append_layer(layer, k, v, i32([lo] * b))
            # the float32 cache takes over all rows' values (an open block's are coded once it fills)
            gk, gv = c.read_rows(layer, i32([0] * b), i32([hi] * b), hi)
            f.append_layer(layer, gk, gv, i32([0] * b))
        for x in (c, f):
            x.commit([hi - lo] * b)

    cfg = CompressionConfig(bits, keep)
    grow(0, n)
    mirrors = [CompressedKVCache(L, cfg, device=dev) for _ in range(2)]
    for m, full in zip(mirrors, (c, f)):
        m.sync_from(full, 0)

    def same():
        for layer in range(L):
            for s in range(b):
                x, y = (m.read_codes(layer, s) if bits < 16 else dict(zip("kvp", m.read(layer, s))) for m in mirrors)
                for key in x:
                    assert np.array_equal(x[key], y[key]), (layer, s, key)

    same()
    grow(n, n + 20)
    for m, full in zip(mirrors, (c, f)):
        m.sync_from(full, n - 3)
    same()
    for m, full in zip(mirrors, (c, f)):
        m.rebuild_layers(full, [1])
    same()


@pytest.mark.gpu
@pytest.mark.parametrize("family,dtype", [("llama", F32), ("tiny", F32), ("llama", BF16)])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_engine_over_it_is_lossless(dev, family, dtype, temperature):
    """Greedy speculative decoding over an 8-bit full cache gives plain decoding's tokens over one, single and batched
    prompts; sampling runs."""
    from draftkv import CompressionConfig, DraftKVEngine, FixedPolicy
    from draftkv.llama import demo_llama
    from draftkv.model import demo_model
    model = demo_llama(dtype=dtype, device=dev) if family == "llama" else demo_model(device=dev)
    model.kv_dtype = F8
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 128, size=n).tolist() for n in (5, 33, 130)]
    for arm, gamma in ((CompressionConfig(4, 0.5), 4), (CompressionConfig(8, 1.0), 7), (CompressionConfig(4, 0.5), 0)):
        eng = DraftKVEngine(model, FixedPolicy(arm, gamma), seed=3)
        got = [r.tokens for r in eng.generate_batch(prompts, 40, temperature)]
        assert eng.last_full.fp8
        if temperature == 0.0:
            assert got == DraftKVEngine(model, seed=3).generate_baseline_batch(prompts, 40)
            assert got[1] == DraftKVEngine(model, FixedPolicy(arm, gamma)).generate(prompts[1], 40).tokens
        else:
            assert all(len(t) == len(p) + 40 for t, p in zip(got, prompts))


@pytest.mark.gpu
@pytest.mark.parametrize("tail,most", [(32, 1), (48, 17)])
def test_the_engine_drafts_no_more_than_the_tail_takes_back(dev, tail, most):
    from draftkv import CompressionConfig, DraftKVEngine, FixedPolicy
    from draftkv.engine import DecodeBatch
    from draftkv.llama import demo_llama
    model = demo_llama(dtype=F32, device=dev)
    model.kv_dtype = F8
    prompts = [np.random.default_rng(s).integers(0, 128, size=n).tolist() for s, n in ((0, 30), (1, 49))]
    want = DraftKVEngine(model).generate_baseline_batch([list(p) for p in prompts], 60)
    eng = DraftKVEngine(model, FixedPolicy(CompressionConfig(2, 0.3), 20))
    full = model.new_cache(2, 200, tail_rows=tail)
    assert full.tail_rows == tail and full.max_rollback == most
    eng._prefill(prompts, full)
    batch = DecodeBatch(eng, prompts, full, 60, 0.0)
    while batch.step():
        pass
    res = batch.results()
    assert [r.tokens for r in res] == want
    gammas = [r.gamma for r in res[0].rounds]
    assert max(gammas) == most


@pytest.mark.gpu
@pytest.mark.parametrize("bs,tail,D,H", [(16, 32, 64, 2), (16, 128, 24, 1), (64, 96, 128, 1), (128, 144, 256, 1), (32, 64, 192, 1)])
def test_appends_made_again(dev, bs, tail, D, H):
    """An append that is not committed may be made again from the same start, or another one in its place, however long:
    the rows before it are there (its open block's, whose places in the tail a long append takes, too)."""
    g = torch.Generator(device=dev)
    g.manual_seed(bs + D)
    rng = np.random.default_rng(bs + tail + D)
    size = 900
    c = new_cache(H, D, bs, size, tail_rows=tail)
    c.reserve([size])
    k, v = rows_of(g, 1, size, H, D, dev)      # the rows that are there, [0, n)
    n, left = 0, 0                              # left: the first row that the tail still holds

    def check(n):
        gk, gv = c.read_rows(0, i32([0]), i32([n]), n + 1)
        for got, x in ((gk, k), (gv, v)):
            assert torch.equal(got[0, :n].double().cpu(), values(x[0, :n].to(BF16).cpu(), bs)), n

    def append(T, fresh):
        nonlocal k, v
        if fresh:                               # other rows from n on
            k2, v2 = rows_of(g, 1, T, H, D, dev)
            k[:, n:n + T], v[:, n:n + T] = k2, v2
        q = torch.randn(1, T, H, D, generator=g, device=dev)
        return [c.append_attend(0, q, k[:, n:n + T].contiguous(), v[:, n:n + T].contiguous(), i32([n]), n + T) for _ in range(2)]

    for _ in range(40):
        if n > 500:                             # another sequence in this one's place
            n = left = 0
        for again in range(int(rng.integers(1, 4))):
            T = int(rng.choice([1, 3, 17, tail - bs + 2, tail + 5, tail + 2 * bs + 9]))
            a, b = append(T, again > 0)
            assert torch.equal(a, b), (n, T)
            check(n)
            left = max(left, min(-(-(n + T) // 16) * 16 - tail, n // bs * bs))
        n += T
        left = max(left, -(-n // 16) * 16 - tail)
        check(n)
        if rng.random() < 0.4:                  # a rollback, within the rows that are left or to a block's end
            cut = int(rng.integers(max(n - 20, 0), n + 1))
            n = cut if cut // bs * bs >= left else cut // bs * bs
            left = min(left, n)
            check(n)


@pytest.mark.gpu
def test_a_forward_that_fails_leaves_the_cache_as_it_was(dev, monkeypatch):
    """A long forward that fails after some layers took its rows: what the cache holds, the mirror from it and the forward
    that follows are those of a cache that never saw it; rollbacks past the open block are refused, its rows are gone."""
    from draftkv import CompressionConfig
    from draftkv.compress import CompressedKVCache
    from draftkv.llama import demo_llama
    model = demo_llama(dtype=F32, device=dev)
    model.kv_dtype = F8
    toks = np.random.default_rng(5).integers(0, 128, size=500)
    full, ref = model.new_cache(max_tokens=1000), model.new_cache(max_tokens=1000)
    for c in (full, ref):
        model.forward(toks[:100], c, 0)
        model.forward(toks[100:150], c, 100)
    calls = 0
    real = model._mlp_inner

    def fails(x, p):
        nonlocal calls
        calls += 1
        if calls == 2:
            raise MemoryError("out of memory")
        return real(x, p)

    monkeypatch.setattr(model, "_mlp_inner", fails)
    with pytest.raises(MemoryError):
        model.forward(toks[150:450], full, 150)
    monkeypatch.undo()
    assert full.length == 150
    for L in range(model.n_layers):
        for a, b in zip(full.read(L), ref.read(L)):
            assert np.array_equal(a, b)
    mirrors = [CompressedKVCache(model.n_layers, CompressionConfig(8, 1.0), device=dev) for _ in range(2)]
    for start in (0, 130):
        for m, c in zip(mirrors, (full, ref)):
            m.sync_from(c, start)
        for L in range(model.n_layers):
            for a, b in zip(mirrors[0].read(L), mirrors[1].read(L)):
                assert np.array_equal(a, b)
    with pytest.raises(ValueError, match="gone"):
        full.truncate(143)                  # rows 128 .. 143 were in the tail before, 144 on are the open block
    for lo, hi in ((150, 155), (155, 450)):
        assert np.array_equal(model.forward(toks[lo:hi], full, lo), model.forward(toks[lo:hi], ref, lo))
    full.truncate(445)
    ref.truncate(445)
    assert np.array_equal(model.forward(toks[445:446], full, 445), model.forward(toks[445:446], ref, 445))


# ---------------------------------------------------------------- refusals (no GPU)
def _desc(**kw):
    from draftkv import _lib
    a = dict(pool=16, block_table=16, tail=16, hot=None, batch=1, n_layers=1, n_kv_heads=2, head_dim=64, block_size=16,
             max_blocks=4, tail_rows=128, hot_rows=0)
    return _lib.Paged8(**{**a, **kw})


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers: host checks only")
@pytest.mark.parametrize("kw,word", [
    (dict(pool=None), "NULL"), (dict(block_table=None), "NULL"), (dict(tail=None), "NULL"), (dict(head_dim=257), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(block_size=24), "block_size"), (dict(block_size=256), "block_size"),
    (dict(tail_rows=16), "tail_rows"), (dict(tail_rows=100), "tail_rows"), (dict(batch=0), "shape"),
    (dict(n_kv_heads=70000), "too many"), (dict(pool=24), "aligned")])
def test_bad_caches_are_refused(kw, word):
    import ctypes as C
    from draftkv import _lib
    L, d = _lib.lib(), _desc(**kw)
    for rc in (L.dkv_paged8_append(C.byref(d), 0, 16, 16, 0, 1, 16, None, None),
               L.dkv_paged8_attention(C.byref(d), 0, 16, 0, 1, 2, 16, None, 64, 16, 16, 1 << 30, None),
               L.dkv_paged8_read(C.byref(d), 0, 16, 16, 1, 16, 16, None)):
        assert rc == -1 and word in L.dkv_last_error().decode()


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers: host checks only")
def test_bad_calls_are_refused():
    import ctypes as C
    from draftkv import _lib
    L, d = _lib.lib(), _desc()

    def err(rc, code, word):
        assert rc == code and word in L.dkv_last_error().decode(), (rc, L.dkv_last_error())

    r = C.byref(d)
    err(L.dkv_paged8_append(r, 1, 16, 16, 0, 1, 16, None, None), -1, "layer")
    err(L.dkv_paged8_append(r, 0, None, 16, 0, 1, 16, None, None), -1, "NULL")
    err(L.dkv_paged8_append(r, 0, 16, 16, 2, 1, 16, None, None), -1, "dtype")
    err(L.dkv_paged8_append(r, 0, 16, 16, 0, 114, 16, None, None), -3, "hot rows")
    err(L.dkv_paged8_attention(r, 0, 16, 0, 114, 2, 16, None, 64, 16, 16, 1 << 30, None), -3, "hot rows")
    err(L.dkv_paged8_attention(r, 0, 16, 2, 1, 2, 16, None, 64, 16, 16, 1 << 30, None), -1, "dtype")
    err(L.dkv_paged8_attention(r, 0, 16, 0, 1, 3, 16, None, 64, 16, 16, 1 << 30, None), -1, "multiple")
    err(L.dkv_paged8_attention(r, 0, 16, 0, 1, 2, 16, None, 0, 16, 16, 1 << 30, None), -1, "max_len")
    err(L.dkv_paged8_attention(r, 0, 16, 0, 1, 2, 16, None, 4096, 16, 16, 64, None), -3, "workspace")
    err(L.dkv_paged8_attention(r, 0, 16, 0, 1, 2, 16, None, 4096, 16, None, 1 << 30, None), -3, "workspace")
    err(L.dkv_paged8_attention(r, 0, 16, 0, 1, 2, None, None, 64, 16, 16, 1 << 30, None), -1, "NULL")
    err(L.dkv_paged8_read(r, 0, 16, None, 1, 16, 16, None), -1, "NULL")
    assert L.dkv_paged8_append(r, 0, 16, 16, 0, 0, 16, None, None) == 0
    assert L.dkv_paged8_hot_rows(r, 113) == 0 and L.dkv_paged8_hot_rows(r, 114) == 144


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers: host checks only")
def test_held_rows_are_checked():
    import ctypes as C
    from draftkv import _lib
    L, d = _lib.lib(), _desc(held=24)
    assert L.dkv_paged8_append(C.byref(d), 0, 16, 16, 0, 1, 16, None, None) == -1 and "held" in L.dkv_last_error().decode()
    for kw, tile in ((dict(head_dim=64), 4096 + 16), (dict(head_dim=8), 2048 + 16), (dict(head_dim=200, block_size=32), 16384 + 32)):
        d = _desc(batch=3, n_layers=5, **kw)
        assert L.dkv_paged8_held_bytes(C.byref(d)) == 3 * 5 * 2 * d.block_size // 16 * tile
    assert L.dkv_paged8_held_bytes(None) == 0 and L.dkv_paged8_held_bytes(C.byref(_desc(head_dim=0))) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers: host checks only")
def test_sizes_past_the_plans_are_refused():
    import ctypes as C
    from draftkv import _lib
    L, top = _lib.lib(), 65534 * 2048
    for max_len in (top + 1, 2 ** 31 - 2048, 2 ** 31 - 1):
        assert L.dkv_paged8_attention(C.byref(_desc()), 0, 16, 0, 1, 2, 16, None, max_len, 16, 16, 1 << 62, None) == -1
        assert "max_len" in L.dkv_last_error().decode()
        assert L.dkv_paged8_attention_workspace(C.byref(_desc()), 1, 2, max_len) == 0
    assert L.dkv_paged8_attention_workspace(C.byref(_desc()), 1, 2, top) > 0
    for D in (257, 500, 2 ** 31 - 1):
        assert L.dkv_paged8_attention_workspace(C.byref(_desc(head_dim=D)), 300, 2, 9000) == 0


def test_tensors_on_another_device_are_refused():
    from draftkv.paged import PagedKVCache
    c = PagedKVCache(1, 2, 64, 16, 4, F8, device="cpu")
    k, st = torch.zeros(1, 1, 2, 64, device="meta"), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: c.append_layer(0, k, k, st), lambda: c.attend(0, k, st, 16), lambda: c.append_attend(0, k, k, k, st, 16),
                 lambda: c.read_rows(0, st.to("meta"), st, 1)):
        with pytest.raises(ValueError, match="for a cache on"):
            call()


def test_bad_constructions_are_refused():
    from draftkv.paged import PagedKVCache
    for kw, word in ((dict(block_size=48), "block_size"), (dict(d_head=300), "d_head"), (dict(tail_rows=20), "tail_rows")):
        a = dict(n_layers=1, n_heads=2, d_head=64, block_size=16, n_blocks=4, dtype=F8, device="cpu")
        with pytest.raises(ValueError, match=word):
            PagedKVCache(**{**a, **kw})
    c = PagedKVCache(1, 2, 64, 16, 4, F8, device="cpu")
    with pytest.raises(ValueError, match="GPU tensor"):
        c.attend(0, torch.zeros(1, 1, 4, 64), torch.zeros(1, dtype=torch.int32), 16)
    with pytest.raises(ValueError, match="8-bit"):
        PagedKVCache(1, 2, 64, 16, 4, torch.float32, device="cpu").read_rows(0, None, None, 1)
