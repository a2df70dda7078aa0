"""Microscaled 4-bit floating point: quantization, products and models with 4-bit weights, against the definition
(OCP MX 1.0, MXFP4) in 64 bits."""

import math

import numpy as np
import pytest
import torch

F32, F64, BF16, F8 = torch.float32, torch.float64, torch.bfloat16, torch.float8_e4m3fn
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def held(x):
    """x [rows, k]: the float64 values its 4-bit form stands for. Nearest of the grid, ties to the even code."""
    r, k = x.shape
    x = torch.cat([x.double().cpu(), torch.zeros(r, -k % 32, dtype=F64)], 1).view(r, -1, 32)
    amax = x.abs().amax(-1)
    e = torch.zeros_like(amax)
    ok = (amax > 0) & torch.isfinite(amax)
    ex = torch.frexp(torch.where(ok, amax, torch.ones_like(amax)))[1].double()
    e = torch.where(ok, torch.clamp(ex - 1 - 2, min=-126), e)
    y = (x / torch.exp2(e)[..., None]).abs()
    g = torch.tensor(GRID, dtype=F64)
    mid = (g[1:] + g[:-1]) / 2
    code = torch.bucketize(y, mid)                       # mid[i-1] < y <= mid[i]: a tie goes down ...
    tie = (y[..., None] == mid).any(-1)
    code = torch.where(tie & (code % 2 == 1), code + 1, code)   # ... or up, to the even code
    v = g[code.clamp(max=7)] * torch.sign(x) * torch.exp2(e)[..., None]
    v = torch.where(torch.isfinite(amax)[..., None], v, torch.full_like(v, math.nan))
    return v.reshape(r, -1)[:, :k]


def same(got, want):
    return torch.equal(torch.nan_to_num(got.double().cpu(), nan=77.0), torch.nan_to_num(want, nan=77.0))


# ---------------------------------------------------------------- quantize
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (16, 128), (17, 576), (5, 100), (33, 1000), (3, 4096), (200, 129), (1, 5001), (130, 31)])
def test_quantize_and_values(dev, rows, k, dtype):
    from draftkv import ops
    g = torch.Generator(device=dev)
    g.manual_seed(rows + k)
    x = (torch.randn(rows, k, generator=g, device=dev) * torch.exp(3 * torch.randn(rows, 1, generator=g, device=dev))).to(dtype)
    x[0, : min(k, 40)] = 0
    q, v = ops.mx4_quantize(x, values=True)
    want = held(x)
    assert q.shape == (rows, k) and same(v, want) and same(q.values(), want)
    assert torch.equal(ops.mx4_quantize(x).codes, q.codes)


@pytest.mark.gpu
def test_quantize_ties_and_extremes(dev):
    from draftkv import ops
    x = torch.zeros(12, 64, device=dev)
    x[0, :16] = torch.tensor([4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, 7.9])   # ties, saturation
    x[1, 32:] = 2.0 ** -140 * torch.arange(32)            # below 2^-126
    x[2] = 3.4e38
    x[3, 5] = math.nan
    x[4, 40] = -math.inf
    x[5, :4] = torch.tensor([1.0, 1e-30, -1e-45, 0.0])
    x[6] = -1e-38
    x[7] = 2.0 ** torch.arange(64) / 2 ** 40
    for t in (x, x.to(BF16)):
        q, v = ops.mx4_quantize(t, values=True)
        want = held(t)
        assert same(v, want) and same(q.values(), want)
        assert v[3, :32].isnan().all() and v[4, 32:].isnan().all() and not v[3, 32:].isnan().any()


# ---------------------------------------------------------------- product
def tol(x, w, dtype, want):
    """Every product is exact in float32 (8 and 2 bits, or 2 and 2); a sum of K of them, in any order, is off by at
    most K steps of half an ulp of the sum of magnitudes. bf16 out: half a step of the result, 2^-8 of it."""
    t = x.shape[1] * 2.0 ** -24 * (x.abs() @ w.abs().t())
    return t if dtype == F32 else t + 2.0 ** -8 * want.abs()


SIZES = [(1, 16, 32), (1, 960, 576), (3, 17, 100), (16, 100, 128), (17, 64, 640), (33, 250, 1000), (64, 48, 4096), (65, 1030, 257),
         (160, 512, 512), (130, 33, 2304), (300, 768, 768), (2, 5, 1), (4096, 1021, 384), (200, 4099, 512), (90, 16390, 256), (700, 257, 128), (1, 20000, 96), (70, 9000, 160),
         (1, 64, 640), (12, 90, 200), (20, 100, 4224), (100, 130, 10112), (30, 8200, 256), (50, 8210, 130), (2100, 4099, 640), (330, 16402, 256),
         (250, 33002, 384), (640, 33002, 256), (300, 49000, 128), (75, 33002, 640), (150, 50257, 128), (240, 40004, 128), (700, 8192, 256), (640, 33000, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("xk", ["f32", "bf16", "mx4"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_against_64_bits(dev, M, N, K, xk):
    from draftkv import ops
    g = torch.Generator(device=dev)
    g.manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g, device=dev).to(BF16 if xk == "bf16" else F32)
    w = ops.mx4_quantize(0.05 * torch.randn(N, K, generator=g, device=dev))
    bias = torch.randn(N, generator=g, device=dev)
    xin = ops.mx4_quantize(x) if xk == "mx4" else x
    x64 = xin.values().double() if xk == "mx4" else x.to(BF16).double()
    w64 = w.values().double()
    want = x64 @ w64.t()
    for dtype in (F32, BF16):
        out = ops.gemm_mx4(xin, w, out_dtype=dtype)
        assert out.dtype == dtype and out.shape == (M, N)
        assert ((out.double() - want).abs() <= tol(x64, w64, dtype, want)).all()
    for b in (bias, bias.to(BF16)):
        wb = want + b.double()
        out = ops.gemm_mx4(xin, w, b, out_dtype=F32)
        assert ((out.double() - wb).abs() <= tol(x64, w64, F32, wb) + 2.0 ** -24 * wb.abs()).all()
    if N % 2 == 0:
        # silu(g) u of g, u off by t: |d/dg| <= 1.1 |u|, |d/du| <= |g| + 0.3, and a few roundings
        t = tol(x64, w64, F32, want)
        gt, up, tg, tu = want[:, 0::2], want[:, 1::2], t[:, 0::2], t[:, 1::2]
        ws = gt * torch.sigmoid(gt) * up
        slack = 1.1 * up.abs() * tg + (gt.abs() + 0.3) * tu + 1.1 * tg * tu + 2.0 ** -20 * ws.abs()
        assert ((ops.gemm_mx4(xin, w, out_dtype=F32, swiglu=True).double() - ws).abs() <= slack).all()
        assert ((ops.gemm_mx4(xin, w, swiglu=True).double() - ws).abs() <= slack + 2.0 ** -8 * ws.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("xk", ["f32", "bf16", "mx4"])
@pytest.mark.parametrize("N,K", [(960, 576), (4096, 1024), (6144, 640), (20000, 512), (256, 14336), (50, 100)])
def test_rows_do_not_depend_on_how_many_there_are(dev, N, K, xk):
    from draftkv import ops
    g = torch.Generator(device=dev)
    g.manual_seed(N)
    M = 700
    x = torch.randn(M, K, generator=g, device=dev).to(BF16 if xk == "bf16" else F32)
    w = ops.mx4_quantize(0.05 * torch.randn(N, K, generator=g, device=dev))
    f = (lambda t: ops.gemm_mx4(ops.mx4_quantize(t), w, out_dtype=F32)) if xk == "mx4" else (lambda t: ops.gemm_mx4(t, w, out_dtype=F32))
    ref = f(x)
    for lo, hi in ((0, 1), (699, 700), (3, 19), (5, 38), (10, 74), (0, 130), (200, 456), (100, 613)):
        assert torch.equal(f(x[lo:hi].contiguous()), ref[lo:hi]), (lo, hi)


@pytest.mark.gpu
@pytest.mark.parametrize("xk", ["bf16", "mx4"])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_a_block_that_is_not_finite_is_nan(dev, M, xk):
    from draftkv import ops
    w = torch.randn(64, 256, device=dev)
    w[5, 70] = math.nan
    w[9, 200] = math.inf
    x = torch.randn(M, 256, device=dev)
    q = ops.mx4_quantize(w)
    y = ops.gemm_mx4(ops.mx4_quantize(x) if xk == "mx4" else x.to(BF16), q, out_dtype=F32)
    bad = y.isnan().all(0)
    assert bad[5] and bad[9] and int(y.isnan().any(0).sum()) == 2
    x[0, 3] = math.inf
    y = ops.gemm_mx4(ops.mx4_quantize(x) if xk == "mx4" else x.to(BF16), q, out_dtype=F32)
    assert not torch.isfinite(y[0]).any()
    if M > 1:
        assert torch.isfinite(y[1:, [c for c in range(64) if c not in (5, 9)]]).all()


@pytest.mark.gpu
def test_misaligned_rows_and_empty_products(dev):
    from draftkv import ops
    w = ops.mx4_quantize(torch.randn(40, 96, device=dev))
    buf = torch.randn(10 * 96 + 1, device=dev)
    x = buf[1:].view(10, 96)                       # 4-byte aligned
    assert torch.equal(ops.gemm_mx4(x, w), ops.gemm_mx4(x.clone(), w))
    xb = buf.to(BF16)[1:].view(10, 96)             # 2-byte aligned
    assert torch.equal(ops.gemm_mx4(xb, w), ops.gemm_mx4(xb.clone(), w))
    assert torch.equal(ops.mx4_quantize(x).codes, ops.mx4_quantize(x.clone()).codes)
    assert ops.gemm_mx4(x[:0], w).shape == (0, 40) and ops.mx4_quantize(x[:0]).shape == (0, 96)


@pytest.mark.gpu
def test_stream_and_graph_replays(dev):
    from draftkv import ops
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    w = ops.mx4_quantize(torch.randn(512, 768, generator=g, device=dev))
    xs = [torch.randn(20, 768, generator=g, device=dev) for _ in range(5)]
    x = xs[0].clone()

    def step():
        return ops.gemm_mx4(x, w), ops.gemm_mx4(ops.mx4_quantize(x), w, out_dtype=F32)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, t in enumerate(xs):
        x.copy_(t)
        want = step()
        if i == 0:
            assert all(torch.equal(a, b) for a, b in zip(warm, want))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_graphs_and_streams_do_not_share_scratch(dev):
    """Two graphs recorded one after another and two streams, at once, each with products that pack their rows and add
    chunks through memory; a larger call in between."""
    from draftkv import ops
    g = torch.Generator(device=dev)
    g.manual_seed(2)
    w = ops.mx4_quantize(torch.randn(1000, 8192, generator=g, device=dev))
    xs = [torch.randn(24, 8192, generator=g, device=dev) for _ in range(2)]
    want = [ops.gemm_mx4(x, w, out_dtype=F32) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([ops.gemm_mx4(x, w, out_dtype=F32) for _ in range(8)])
        graphs.append(graph)
    ops.gemm_mx4(torch.randn(900, 8192, generator=g, device=dev), w)      # more scratch than before
    junk = [torch.full((1 << 22,), math.nan, device=dev) for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, ref in zip(outs, want):
            assert all(torch.equal(t, ref) for t in o)
        eager = []
        for i in range(16):
            with torch.cuda.stream(streams[i % 2]):
                eager.append(ops.gemm_mx4(xs[i % 2], w, out_dtype=F32))
        torch.cuda.synchronize()
        assert all(torch.equal(t, want[i % 2]) for i, t in enumerate(eager))
    assert all(t.isnan().all() for t in junk)


@pytest.mark.gpu
@pytest.mark.parametrize("xk", ["bf16", "f32", "mx4"])
def test_rows_past_32_bits_of_bytes(dev, xk):
    from draftkv import ops
    g = torch.Generator(device=dev)
    g.manual_seed(5)
    M, N, K = 150000, 48, 16384          # x: 4.9 GB of bf16
    x = torch.empty(M, K, device=dev, dtype=F32 if xk == "f32" else BF16).normal_(generator=g)
    w = ops.mx4_quantize(torch.randn(N, K, generator=g, device=dev))
    q = ops.mx4_quantize(x) if xk == "mx4" else x
    out = ops.gemm_mx4(q, w, out_dtype=F32)
    for lo in (0, 65536, 131071, 149984):
        part = x[lo:lo + 16].contiguous()
        pq = ops.mx4_quantize(part) if xk == "mx4" else part
        assert torch.equal(ops.gemm_mx4(pq, w, out_dtype=F32), out[lo:lo + 16]), lo
    if xk == "mx4":
        v = ops.MX4(q.codes, q.scales, (M, K)).values()
        assert torch.equal(v[-16:], pq.values())


# ---------------------------------------------------------------- models
@pytest.mark.gpu
@pytest.mark.parametrize("family,dtype", [("llama", F32), ("llama", BF16), ("bias", F32), ("gpt2", F32), ("gpt2", BF16), ("tiny", F32)])
def test_model_with_4_bit_weights(dev, family, dtype):
    """Its logits are those of the same model with the values that the 4-bit weights stand for (bf16 activations aside),
    and greedy speculative decoding equals plain decoding, over the model's own and over an 8-bit full cache."""
    from draftkv import CompressionConfig, DraftKVEngine, FixedPolicy, FullKVCache
    from draftkv.gpt2 import GPT2
    from draftkv.llama import demo_llama
    from draftkv.model import demo_model

    def make(t):
        if family == "tiny":
            return demo_model(dtype=t, device=dev)
        if family == "gpt2":
            return GPT2.random(dict(n_layer=2, n_head=4, n_embd=64, n_positions=256, vocab_size=128), seed=1, std=0.1, dtype=t, device=dev)
        return demo_llama(attn_bias=family == "bias", dtype=t, device=dev)

    model, plain = make(dtype), make(F32)
    model.quantize_weights()
    for p, q in zip(plain.layers, model.layers):
        for name in ("wqkv", "wo", "w1", "w2"):
            v = getattr(q, name).values()
            if name == "w1" and plain.mlp == "swiglu":
                v = torch.cat([v[0::2], v[1::2]])
            if dtype == F32:
                w = getattr(p, name) if plain.layout == 1 else getattr(p, name).t()
                assert same(v, held(w) if name != "w1" or plain.mlp != "swiglu" else held(w))
            setattr(p, name, v if plain.layout == 1 else v.t().contiguous())
    toks = np.random.default_rng(2).integers(0, 128, size=50)
    got, want = model.forward(toks, model.new_cache(), 0), plain.forward(toks, plain.new_cache(), 0)
    # both operands of a product are exact but for x's rounding to bf16 (2^-8 of each value), through 2 to 4 layers of
    # four products whose logits reach top; bf16 models round every activation as well
    assert np.abs(got - want).max() <= (0.1 if dtype == F32 else 0.3) * np.abs(want).max()
    prompts = [np.random.default_rng(s).integers(0, 128, size=n).tolist() for s, n in ((0, 7), (1, 40))]
    for kv in (model.kv_dtype, F8):
        model.kv_dtype = kv
        got = [r.tokens for r in DraftKVEngine(model, FixedPolicy(CompressionConfig(4, 0.5), 4)).generate_batch(prompts, 30)]
        assert got == DraftKVEngine(model).generate_baseline_batch(prompts, 30)


@pytest.mark.gpu
@pytest.mark.parametrize("family,dtype", [("llama", F32), ("llama", BF16), ("bias", F32), ("bias", BF16), ("gpt2", F32), ("gpt2", BF16), ("tiny", F32)])
def test_model_with_4_bit_weights_step_by_step(dev, family, dtype, monkeypatch):
    """The same model with the 4-bit weights' values, every projection's input rounded to bf16: the products' operands
    are then equal, and the logits differ by the order of float32 sums alone."""
    from draftkv import ops
    from draftkv.gpt2 import GPT2
    from draftkv.llama import demo_llama
    from draftkv.model import demo_model

    def make():
        if family == "tiny":
            return demo_model(dtype=dtype, device=dev)
        if family == "gpt2":
            return GPT2.random(dict(n_layer=2, n_head=4, n_embd=64, n_positions=256, vocab_size=128), seed=1, std=0.1, dtype=dtype, device=dev)
        return demo_llama(attn_bias=family == "bias", dtype=dtype, device=dev)

    model, plain = make(), make()
    for m in (model, plain):                                   # (biases that a logit shows)
        for i, p in enumerate(m.layers):
            for name in ("bqkv", "bo", "b1", "b2"):
                if getattr(p, name) is not None:
                    getattr(p, name).normal_(0.0, 0.5, generator=torch.Generator(device=dev).manual_seed(i))
    model.quantize_weights()
    for p, q in zip(plain.layers, model.layers):
        for name in ("wqkv", "wo", "w1", "w2"):
            v = getattr(q, name).values().to(dtype)            # (exact)
            if name == "w1" and plain.mlp == "swiglu" and not getattr(plain, "gate_up_interleaved", False):
                v = torch.cat([v[0::2], v[1::2]])
            setattr(p, name, v if plain.w_layout == 1 else v.t().contiguous())
    if dtype == F32:
        f, g = ops.gemm_f32, ops.gemm_f32_act
        monkeypatch.setattr(ops, "gemm_f32", lambda x, w, *a, **k: f(x if w is plain.head else x.to(BF16).float(), w, *a, **k))
        monkeypatch.setattr(ops, "gemm_f32_act", lambda x, *a, **k: g(x.to(BF16).float(), *a, **k))
    elif plain.mlp == "swiglu":       # of the float32 gate and up, as the 4-bit product's is (the bf16 one rounds them first)
        def mlp(x, p):
            y = ops.gemm_bf16(x, p.w1, out_dtype=F32)
            gate, up = (y[:, 0::2], y[:, 1::2]) if getattr(plain, "gate_up_interleaved", False) else y.chunk(2, 1)
            return (torch.nn.functional.silu(gate) * up).to(BF16)
        monkeypatch.setattr(plain, "_mlp_inner", mlp)
    toks = np.random.default_rng(2).integers(0, 128, size=50)
    want = plain.forward(toks, plain.new_cache(), 0)
    monkeypatch.undo()
    got = model.forward(toks, model.new_cache(), 0)
    # Sums in another order differ by about 2^-22 of a value, which now and then (2^-22 / 2^-8) puts an activation on the
    # other side of a bf16 step: one of 64 or more inputs of a product by 2^-8 of it, about 2^-11 of the output. A few
    # such per token: 2^-8 of the largest logit. bf16 models round every output as well, a few more: 2^-7.
    assert np.abs(got - want).max() <= (2.0 ** -8 if dtype == F32 else 2.0 ** -7) * np.abs(want).max()


@pytest.mark.gpu
@pytest.mark.parametrize("xk", ["f32", "bf16", "mx4"])
@pytest.mark.parametrize("M,N,K", [(1, 131072, 128), (2, 140001, 40), (70, 131090, 96)])
def test_few_rows_of_very_wide_weights(dev, M, N, K, xk):
    from draftkv import ops
    g = torch.Generator(device=dev)
    g.manual_seed(N)
    x = torch.randn(M, K, generator=g, device=dev).to(BF16 if xk == "bf16" else F32)
    w = ops.mx4_quantize(0.05 * torch.randn(N, K, generator=g, device=dev))
    xin = ops.mx4_quantize(x) if xk == "mx4" else x
    x64, w64 = xin.values().double() if xk == "mx4" else x.to(BF16).double(), w.values().double()
    want = x64 @ w64.t()
    assert ((ops.gemm_mx4(xin, w, out_dtype=F32).double() - want).abs() <= tol(x64, w64, F32, want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("xk", ["f32", "bf16", "mx4"])
@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("ew,ex", [(-128, 100), (-126, 120), (110, -120), (-124, 90)])
def test_products_of_tiny_and_large_values(dev, M, ew, ex, xk):
    """Weights whose values are no normal bf16 numbers, or near the largest, and rows that bring the products back."""
    from draftkv import ops
    g = torch.Generator(device=dev)
    g.manual_seed(ew + 200)
    N, K = 96, 256
    x = (torch.randn(M, K, generator=g, device=dev) * 2.0 ** ex).to(BF16 if xk == "bf16" else F32)
    w = ops.mx4_quantize(torch.randn(N, K, generator=g, device=dev) * 2.0 ** (ew / 2) * 2.0 ** (ew / 2))
    xin = ops.mx4_quantize(x) if xk == "mx4" else x
    x64, w64 = xin.values().double() if xk == "mx4" else x.to(BF16).double(), w.values().double()
    assert w64.any() and torch.isfinite(w64).all()
    want = x64 @ w64.t()
    assert ((ops.gemm_mx4(xin, w, out_dtype=F32).double() - want).abs() <= tol(x64, w64, F32, want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("gamma", [0, 4])
def test_weights_quantized_while_decoding(dev, gamma):
    """Recorded steps hold the weights that they were recorded with: after quantize_weights() they are recorded anew."""
    from draftkv import CompressionConfig, DraftKVEngine, FixedPolicy
    from draftkv.engine import DecodeBatch
    from draftkv.llama import demo_llama
    prompts = [np.random.default_rng(s).integers(0, 128, size=n).tolist() for s, n in ((0, 30), (1, 40))]
    runs, graphs = [], 0
    for use in (True, False):
        m = demo_llama(dtype=F32, device=dev)
        eng = DraftKVEngine(m, FixedPolicy(CompressionConfig(4, 0.5), gamma))
        eng.draft_graphs = use
        full = eng._new_full(2, 200)
        eng._prefill(prompts, full)
        batch = DecodeBatch(eng, prompts, full, 60, 0.0)
        for _ in range(6):
            batch.step()
        old = [w for p in m.layers for w in (p.wqkv, p.wo, p.w1, p.w2)]
        m.quantize_weights()
        for w in old:
            w.fill_(math.nan)     # (nothing reads them any more)
        while batch.step():
            pass
        runs.append([r.tokens for r in batch.results()])
        graphs = max(graphs, len(batch._graphs))
    assert runs[0] == runs[1] and graphs >= 2


# ---------------------------------------------------------------- refusals (no GPU)
@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers: host checks only")
def test_bad_calls_are_refused():
    from draftkv import _lib
    L = _lib.lib()

    def err(rc, word):
        assert rc == -1 and word in L.dkv_last_error().decode(), (rc, L.dkv_last_error())

    err(L.dkv_mx4_quantize(None, 0, 4, 32, 16, 16, None, None), "NULL")
    err(L.dkv_mx4_quantize(16, 2, 4, 32, 16, 16, None, None), "dtype")
    err(L.dkv_mx4_quantize(16, 0, 4, 0, 16, 16, None, None), "shape")
    err(L.dkv_mx4_quantize(16, 0, 4, 32, 8, 16, None, None), "aligned")
    err(L.dkv_mx4_values(16, 16, 4, 32, None, None), "NULL")
    good = dict(x=16, xd=0, xs=None, w=16, ws=16, b=None, bd=0, M=4, N=16, K=32, y=16, yd=0, fl=0)

    def gemm(**kw):
        return L.dkv_gemm_mx4(*{**good, **kw}.values(), None, 0, None)

    for kw, word in ((dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(ws=None), "NULL"), (dict(y=None), "NULL"), (dict(xd=3), "dtype"),
                     (dict(xd=2), "scales"), (dict(yd=2), "dtype"), (dict(b=16, bd=2), "bias"), (dict(N=0), "shape"), (dict(K=0), "shape"),
                     (dict(M=-1), "shape"), (dict(fl=8), "flags"), (dict(fl=1, N=15), "SwiGLU"), (dict(fl=1, b=16), "SwiGLU"),
                     (dict(w=24), "aligned"), (dict(ws=18), "aligned"), (dict(y=24), "aligned"), (dict(xd=2, xs=16, x=20), "aligned")):
        err(gemm(**kw), word)
    assert gemm(M=0) == 0
    assert gemm(M=5) == -3 and "workspace" in L.dkv_last_error().decode()
    assert L.dkv_gemm_mx4_workspace(16, 0, 65, 16, 32) == 65 * 256 and L.dkv_gemm_mx4_workspace(16, 1, 65, 16, 128) == 0
    assert L.dkv_mx4_code_bytes(17, 129) == 2 * 2 * 1024 and L.dkv_mx4_scale_bytes(17, 513) == 2 * 2 * 256


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers: host checks only")
@pytest.mark.parametrize("xd,M,N,K", [(1, 4, 16, 1 << 30), (1, 2, 16, (1 << 30) + 8), (1, 2, 1, 2 ** 31 - 1), (0, 3, 16, 2 ** 31 - 8),
                                      (0, 16, 65536, 1 << 24), (1, 400, 64, (1 << 23) + 1)])
def test_widths_past_32_bit_offsets_are_refused(xd, M, N, K):
    from draftkv import _lib
    L = _lib.lib()
    rc = L.dkv_gemm_mx4(16, xd, None, 16, 16, None, 0, M, N, K, 16, 0, 0, 16, 1 << 62, None)
    assert rc == -1 and "K too large" in L.dkv_last_error().decode()


def test_bad_tensors_are_refused():
    from draftkv import ops
    z = torch.zeros(4, 32)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.mx4_quantize(z)
    with pytest.raises(ValueError, match="must be MX4"):
        ops.gemm_mx4(z, z)
    w = ops.MX4(torch.zeros(1024, dtype=torch.uint8), torch.zeros(256, dtype=torch.uint8), (16, 32))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.gemm_mx4(z, w)
    with pytest.raises(ValueError, match="out_dtype"):
        ops.gemm_mx4(w, w, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="disagree"):
        ops.gemm_mx4(ops.MX4(w.codes, w.scales, (16, 64)), w)
    with pytest.raises(ValueError, match="SwiGLU"):
        ops.gemm_mx4(w, ops.MX4(w.codes, w.scales, (15, 32)), swiglu=True)


def test_matrices_of_other_sizes_are_refused():
    from draftkv import ops
    b = lambda n: torch.zeros(n, dtype=torch.uint8)
    ops.MX4(b(2048), b(512), (17, 128))
    for codes, scales in ((b(1024), b(512)), (b(2048), b(256)), (b(4096)[::2], b(512)), (torch.zeros(2048), b(512))):
        with pytest.raises(ValueError, match="contiguous bytes"):
            ops.MX4(codes, scales, (17, 128))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(16, 100, 128), (3, 17, 100), (130, 36, 64), (40, 1028, 256), (50, 260, 2048), (20, 102, 4200), (12, 50, 4100)])
def test_nothing_is_written_past_the_outputs(dev, M, N, K):
    from draftkv import _lib, ops
    q = ops.mx4_quantize(torch.randn(N, K, device=dev))
    x = torch.randn(M, K, device=dev)
    y = torch.full((M * N + 4096,), 5.0, device=dev)
    n = _lib.lib().dkv_gemm_mx4_workspace(x.data_ptr(), 0, M, N, K)
    ws = torch.full((n + 4096,), 7, dtype=torch.uint8, device=dev)
    _lib.check(_lib.lib().dkv_gemm_mx4(x.data_ptr(), 0, None, q.codes.data_ptr(), q.scales.data_ptr(), None, 0, M, N, K, y.data_ptr(),
                                       0, 0, ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream), "dkv_gemm_mx4")
    assert (ws[n:] == 7).all()
    assert (y[M * N:] == 5.0).all() and torch.equal(y[: M * N].view(M, N), ops.gemm_mx4(x, q, out_dtype=F32))
    codes = torch.full((q.codes.numel() + 4096,), 9, dtype=torch.uint8, device=dev)
    scales = torch.full((q.scales.numel() + 4096,), 9, dtype=torch.uint8, device=dev)
    _lib.check(_lib.lib().dkv_mx4_quantize(x.data_ptr(), 0, min(M, N), K, codes.data_ptr(), scales.data_ptr(), None,
                                           torch.cuda.current_stream().cuda_stream), "dkv_mx4_quantize")
    n, m = (f(min(M, N), K) for f in (_lib.lib().dkv_mx4_code_bytes, _lib.lib().dkv_mx4_scale_bytes))
    assert (codes[n:] == 9).all() and (scales[m:] == 9).all()
