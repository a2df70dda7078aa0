"""The operators of many continuations of one prompt: attention over shared pages, copying pages, beam selection.

A case is a dict of plain values; ``kind`` names the operator:

* ``attn``: ``prompts`` prompts of up to ``ctx`` rows, each continued by ``n`` sequences that hold up to ``own`` rows of
  their own beside the prompt's, and ``tokens`` new rows each whose queries attend (``SharedKVCache.attend``): decode (one
  row), verify (a few). The prompts' pages are there once.
* ``copy``: ``pairs`` pages of a store of ``pages`` are copied over others (``ops.paged_copy``): what a beam step does to
  the pages that its beams still fill, and compaction to pages that move. A page holds 16 tokens of all layers.
* ``beam``: the ``k`` best continuations of ``beams`` beams of ``prompts`` prompts over a vocabulary
  (``ops.beam_select``): float64 scores cum + logit - logsumexp(logits), best first, ties to the lowest beam and token.
"""

import math
import os
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "draft-kv_amd"))

DEV = "cuda"
F32, F64, BF16, I32 = torch.float32, torch.float64, torch.bfloat16, torch.int32
# query heads, KV heads, head width, layers, vocabulary of the models that the framework names
MODELS = {"llama3_8b": (32, 8, 128, 32, 128256), "smollm2": (9, 3, 64, 30, 49152), "distilgpt2": (12, 12, 64, 6, 50257)}
BLOCK = 16


def listed():
    return [
        # four samples of a short prompt from a small float32 model: latency counts
        dict(name="attn_samples_small", kind="attn", model="smollm2", prompts=1, n=4, tokens=1, ctx=501, own=33, kv="f32", q="f32"),
        # 32 samples of one 32k prompt, a decode step as the models run it (float32 queries)
        dict(name="attn_samples_32k", kind="attn", model="llama3_8b", prompts=1, n=32, tokens=1, ctx=32700, own=200, kv="bf16", q="f32"),
        # four prompts of 16k with 16 samples each, bf16 queries
        dict(name="attn_samples_4x16", kind="attn", model="llama3_8b", prompts=4, n=16, tokens=1, ctx=16000, own=500, kv="bf16", q="bf16"),
        # the verify pass (gamma 4) of 32 samples of one 32k prompt
        dict(name="attn_verify_32k", kind="attn", model="llama3_8b", prompts=1, n=32, tokens=5, ctx=32700, own=100, kv="bf16", q="f32"),
        # a beam step: eight prompts of different lengths, four beams each
        dict(name="attn_beams", kind="attn", model="llama3_8b", prompts=8, n=4, tokens=1, ctx=4001, own=60, kv="bf16", q="f32"),
        # a float32 cache without grouped heads, three rows each
        dict(name="attn_f32_verify", kind="attn", model="distilgpt2", prompts=2, n=8, tokens=3, ctx=900, own=100, kv="f32", q="f32"),
        # four beams of one prompt, a small vocabulary: latency counts
        dict(name="beam_small", kind="beam", prompts=1, beams=4, vocab=49152, k=8, dtype="f32"),
        # eight prompts of four beams
        dict(name="beam_8x4", kind="beam", prompts=8, beams=4, vocab=128256, k=8, dtype="f32"),
        # a large batch of wide beams
        dict(name="beam_32x8", kind="beam", prompts=32, beams=8, vocab=128256, k=16, dtype="f32"),
        # the open pages of a few beams of a small model
        dict(name="copy_small", kind="copy", model="smollm2", pairs=6, pages=64, dtype="f32"),
        # a beam step of eight prompts of four beams, three of each four moved
        dict(name="copy_beams", kind="copy", model="llama3_8b", pairs=24, pages=200, dtype="bf16"),
        # compaction: pages that move to the front of the pool
        dict(name="copy_compact", kind="copy", model="llama3_8b", pairs=160, pages=500, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "beam", "beam", "copy"])
    if kind == "attn":
        prompts, n = rng.choice([1, 1, 2, 3, 5, 8]), _log(rng, 2, 32)
        return dict(kind=kind, model=rng.choice(["llama3_8b", "llama3_8b", "smollm2", "distilgpt2"]), prompts=prompts, n=n,
                    tokens=rng.choice([1, 1, 1, 2, 3, 5]), ctx=_log(rng, 16, min(32000, 500000 // (prompts * n))),
                    own=_log(rng, 1, 300), kv=rng.choice(["bf16", "bf16", "f32"]), q=rng.choice(["f32", "f32", "bf16"]))
    if kind == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        return dict(kind=kind, prompts=_log(rng, 1, 256 // beams), beams=beams, vocab=rng.choice([1000, 32001, 49152, 50257, 128256]),
                    k=rng.randrange(1, 33), dtype=rng.choice(["f32", "f32", "bf16"]))
    pairs = _log(rng, 1, 128)
    return dict(kind=kind, model=rng.choice(list(MODELS)), pairs=pairs, pages=2 * pairs + rng.randrange(1, 100), dtype=rng.choice(["f32", "bf16"]))


# ---------------------------------------------------------------- inputs
_TYPES = {"f32": F32, "bf16": BF16}


def _lengths(case):
    """Rows of each prompt, and the rows of their own that the sequences hold before the new ones."""
    ctx = [case["ctx"] - 37 * p % (case["ctx"] // 4 + 1) for p in range(case["prompts"])]
    rows = [case["own"] - 5 * s % (case["own"] // 2 + 1) for s in range(case["prompts"] * case["n"])]
    return ctx, rows


def _normal(g, *shape, std=1.0, dtype=F32):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


def _kv(g, b, n, heads, d, dtype):
    """K and V rows [b, n, heads, d]: normal, K with the uneven channel gains that trained models show."""
    gain = torch.exp(0.4 * _normal(g, heads, d)).to(dtype)
    return _normal(g, b, n, heads, d, dtype=dtype).mul_(gain), _normal(g, b, n, heads, d, dtype=dtype)


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "attn":
        hq, h, d = MODELS[case["model"]][:3]
        kv = _TYPES[case["kv"]]
        b, t = case["prompts"] * case["n"], case["tokens"]
        s["ck"], s["cv"] = _kv(g, case["prompts"], case["ctx"], h, d, kv)
        s["k"], s["v"] = _kv(g, b, case["own"] + t, h, d, kv)
        s["q"] = _normal(g, b, t, hq, d, dtype=_TYPES[case["q"]])
    elif case["kind"] == "beam":
        p, b, v = case["prompts"], case["beams"], case["vocab"]
        # a model's logits: a wide bulk, and a few tokens well above it
        x = _normal(g, p, b, v)
        s["x"] = (1.8 * x + 0.12 * x * x * x).to(_TYPES[case["dtype"]])
        s["cum"] = -20.0 * torch.rand((p, b), dtype=F64, device=DEV, generator=g)
        s["cum"][0, 1:] = -math.inf        # the first step of a prompt: one beam lives
    else:
        hq, h, d, layers = MODELS[case["model"]][:4]
        n, pages = case["pairs"], case["pages"]
        s["store"] = _normal(g, pages, layers * 2 * h * BLOCK * d, dtype=_TYPES[case["dtype"]])
        perm = torch.randperm(pages, device=DEV, generator=g)
        # a page may go to several places (a beam with several children); no page is read and written
        s["src"] = perm[n:2 * n][torch.randint(0, n, (n,), device=DEV, generator=g)].to(I32)
        s["dst"] = perm[:n].to(I32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] != "attn" or not own:
        return s
    from draftkv.shared import SharedKVCache
    p, n, t = case["prompts"], case["n"], case["tokens"]
    ctx, rows = _lengths(case)
    h, d = s["k"].shape[2:]
    most = case["ctx"] + case["own"] + t
    pages = sum(-(-c // BLOCK) for c in ctx) + p * n * (-(-(case["own"] + t) // BLOCK) + 1)
    c = SharedKVCache(1, h, d, BLOCK, pages, _TYPES[case["kv"]], batch=p, max_tokens=most, device=DEV)
    c.reserve(ctx)
    c.append_layer(0, s.pop("ck"), s.pop("cv"), torch.zeros(p, dtype=I32, device=DEV), torch.tensor(ctx, dtype=I32, device=DEV))
    c.commit(ctx)
    c.fork([i // n for i in range(p * n)])
    start = torch.tensor([ctx[i // n] for i in range(p * n)], dtype=I32, device=DEV)
    new = [r + t for r in rows]
    c.reserve(new)
    c.append_layer(0, s.pop("k"), s.pop("v"), start, torch.tensor(new, dtype=I32, device=DEV))
    c.commit(new)
    s["cache"] = c
    s["start"] = start + torch.tensor(rows, dtype=I32, device=DEV)
    s["max_len"] = max(ctx[i // n] + new[i] for i in range(p * n))
    return s


# ---------------------------------------------------------------- plain forms
def _attend(s):
    case = s["case"]
    n, t = case["n"], case["tokens"]
    ctx, rows = _lengths(case)
    q = s["q"].float()
    hq, d = q.shape[2:]
    h = s["ck"].shape[2]
    g = hq // h
    out = torch.empty_like(q)
    for p in range(case["prompts"]):
        mine = slice(p * n, (p + 1) * n)
        qq = (q[mine] / math.sqrt(d)).view(n, t, h, g, d).permute(2, 0, 1, 3, 4).contiguous()      # [h, n, t, g, d]
        ck, cv = (s[x][p, : ctx[p]].permute(1, 0, 2).float().contiguous() for x in ("ck", "cv"))    # [h, ctx, d]
        k, v = (s[x][mine].permute(2, 0, 1, 3).float().contiguous() for x in ("k", "v"))            # [h, n, own + t, d]
        sc = qq.view(h, n * t * g, d) @ ck.transpose(1, 2).contiguous()
        so = qq.view(h, n, t * g, d) @ k.transpose(2, 3).contiguous()
        row = torch.tensor(rows[mine], device=DEV).view(n, 1, 1) + torch.arange(t, device=DEV).repeat_interleave(g).view(1, t * g, 1)
        so = torch.where(torch.arange(k.shape[2], device=DEV) <= row, so, -math.inf).view(h, n * t * g, -1)
        m = torch.maximum(sc.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
        sc, so = torch.exp(sc - m), torch.exp(so - m)
        o = sc @ cv + (so.view(h, n, t * g, -1) @ v).view(h, n * t * g, d)
        o = o / (sc.sum(-1, keepdim=True) + so.sum(-1, keepdim=True))
        out[mine] = o.view(h, n, t, g, d).permute(1, 2, 0, 3, 4).reshape(n, t, hq, d)
    return out.to(s["q"].dtype)


def _select(s):
    x = s["x"].double()
    p, b, v = x.shape
    m = x.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    score = (s["cum"][..., None] + (x - lse)).view(p, b * v)
    k = s["case"]["k"]
    best, at = torch.sort(score, dim=-1, descending=True, stable=True)      # equal scores: the lowest beam and token first
    best, at = best[:, :k], at[:, :k]
    none = best == -math.inf
    return [best.contiguous(), torch.where(none, -1, at // v).to(I32), torch.where(none, -1, at % v).to(I32)]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        return _run_own(s, case, kind)
    if kind == "attn":
        return _attend(s)
    if kind == "beam":
        return _select(s)
    s["store"][s["dst"].long()] = s["store"][s["src"].long()]
    return s["store"]


def _run_own(s, case, kind):
    from draftkv import ops
    if kind == "attn":
        return s["cache"].attend(0, s["q"], s["start"], s["max_len"])
    if kind == "beam":
        return list(ops.beam_select(s["x"], s["cum"], case["k"]))
    return ops.paged_copy(s["store"], s["src"], s["dst"])


# ---------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "bf16": 2}
    if case["kind"] == "copy":
        h, d, layers = MODELS[case["model"]][1:4]
        return {"bytes": 2 * case["pairs"] * layers * 2 * h * BLOCK * d * size[case["dtype"]], "flops": 0}
    if case["kind"] == "beam":
        rows = case["prompts"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * size[case["dtype"]] + 8) + case["prompts"] * case["k"] * 16, "flops": 0}
    hq, h, d = MODELS[case["model"]][:3]
    n, t = case["n"], case["tokens"]
    ctx, rows = _lengths(case)
    keys = sum(t * (ctx[i // n] + r) + t * (t + 1) // 2 for i, r in enumerate(rows))    # (row, key) pairs per query head
    held = sum(ctx) + sum(r + t for r in rows)
    return {"bytes": 2 * held * h * d * size[case["kv"]] + 2 * len(rows) * t * hq * d * size[case["q"]], "flops": 4 * hq * d * keys}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "copy":
        want = s["store"].clone()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            want[b] = s["store"][a]
        return want
    if case["kind"] == "beam":
        x = s["x"].to(F64)
        p, b, v = x.shape
        logp = (x - torch.logsumexp(x, -1, keepdim=True) + s["cum"][..., None]).view(p, b * v)
        index = torch.arange(b * v, device=DEV)
        best, parent, token = [], [], []
        for _ in range(case["k"]):
            top = logp.amax(-1, keepdim=True)
            at = torch.where(logp == top, index, b * v).amin(-1)       # the first of the best
            gone = top[:, 0] == -math.inf
            best.append(top[:, 0])
            parent.append(torch.where(gone, -1, at // v))
            token.append(torch.where(gone, -1, at % v))
            logp[torch.arange(p, device=DEV), at] = -math.inf
        return [torch.stack(best, 1), torch.stack(parent, 1).to(I32), torch.stack(token, 1).to(I32)]
    n, t = case["n"], case["tokens"]
    ctx, rows = _lengths(case)
    q = s["q"].to(F64)
    g = q.shape[2] // s["k"].shape[2]
    o = torch.empty_like(q)
    for i, r in enumerate(rows):
        p = i // n
        for j in range(s["k"].shape[2]):
            k, v = (torch.cat([s["c" + x][p, : ctx[p], j], s[x][i, : r + t, j]]).to(F64) for x in "kv")
            qq = q[i, :, j * g:(j + 1) * g]
            sc = (qq.reshape(t * g, -1) @ k.t()).view(t, g, -1) / math.sqrt(k.shape[1])
            seen = torch.arange(k.shape[0], device=DEV) <= (ctx[p] + r + torch.arange(t, device=DEV))[:, None, None]
            w = torch.softmax(torch.where(seen, sc, -math.inf), -1)
            o[i, :, j * g:(j + 1) * g] = (w.reshape(t * g, -1) @ v).view(t, g, -1)
    return o
