"""Captured steps of a prefix that has been replaced are dropped, not kept for good."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch

from leanstack_b200 import synth
from leanstack_b200.config import TINY
from leanstack_b200.engine import DecodeEngine
from leanstack_b200.leanserve import materialize_from_tensors
from leanstack_b200.speculative import SpeculativeDecoder

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def runtime():
    return materialize_from_tensors(TINY, {k: v.to(DEV) for k, v in synth.synth_checkpoint(TINY, 3).items()}, device=DEV)


def _ids(name, *shape):
    return synth.token_ids(shape, TINY.vocab_size, 3, f"stale/{name}")


def test_speculative_cycles(runtime):
    draft, target = (DecodeEngine(runtime, 2, 96, max_tokens_per_step=16, linear_backend="tc", prefix_capacity=30)
                     for _ in range(2))
    spec = SpeculativeDecoder(draft, target, 3, 8)
    graphs = []
    for i in range(4):
        for e in (draft, target):
            e.reset()
            e.prefill_prefix(_ids(f"p{i}", 20 + i))
        spec.generate(_ids("prompt", 2, 7).to(DEV), 8)
        spec.cycle(2)  # another proposal length, the same prefix: beside the first
        assert sorted(k[0] for k in spec.graphs) == [2, 3]
        graphs += [weakref.ref(g) for g in spec.graphs.values()]
        torch.cuda.synchronize()
    gc.collect()
    assert [r() is not None for r in graphs] == [False] * 6 + [True] * 2
