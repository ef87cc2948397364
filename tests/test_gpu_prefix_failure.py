"""A prefix whose pass fails leaves an engine without a prefix: no captured step, seen token or length of the old one."""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import synth
from leanstack_b200.config import TINY
from leanstack_b200.engine import DecodeEngine
from leanstack_b200.leanserve import materialize_from_tensors
from leanstack_b200.requests import TokenRules

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def runtime():
    return materialize_from_tensors(TINY, {k: v.to(DEV) for k, v in synth.synth_checkpoint(TINY, 3).items()}, device=DEV)


def _ids(name, *shape):
    return synth.token_ids(shape, TINY.vocab_size, 3, f"failure/{name}")


def test_a_failed_prefix(runtime, monkeypatch):
    def engine():
        rules = TokenRules(3, TINY.vocab_size, DEV)
        for b in range(3):
            rules.set_request(b, repetition=1.3)
        return DecodeEngine(runtime, 3, 64, prefix_capacity=40, rules=rules), rules

    prompt = _ids("prompt", 3, 6).to(DEV)
    plain, _ = engine()
    want = plain.generate(prompt, 5)
    eng, rules = engine()
    eng.prefill_prefix(_ids("first", 33))
    eng.generate(prompt, 3)  # captures the step
    eng.reset()
    with monkeypatch.context() as m:
        m.setattr(eng, "_prompt_pass", lambda *a: (_ for _ in ()).throw(RuntimeError("out of memory")))
        with pytest.raises(RuntimeError, match="out of memory"):
            eng.prefill_prefix(_ids("second", 40))
    assert eng.prefix_len == 0
    assert not rules.seen.any() and not rules.prefix_seen.any()
    assert torch.equal(eng.generate(prompt, 5), want)
