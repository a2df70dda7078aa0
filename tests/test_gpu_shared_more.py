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
