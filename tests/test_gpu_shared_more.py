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
