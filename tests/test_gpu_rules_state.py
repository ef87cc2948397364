"""What the engine keeps of the token rules: every pick follows from prefix, prompt and answer, batch after batch.

The rules are restated on the CPU from the tokens alone and applied to the engine's own logits, so a token that is
missing from the kernel's state, or left over in it, changes the expected pick or the expected state.
"""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import kernels as K
from leanstack_b200 import synth
from leanstack_b200.config import TINY
from leanstack_b200.engine import DecodeEngine
from leanstack_b200.leanserve import materialize_from_tensors
from leanstack_b200.requests import TokenRules

pytestmark = pytest.mark.gpu
DEV = "cuda"
V = TINY.vocab_size


@pytest.fixture(scope="module")
def runtime():
    return materialize_from_tensors(TINY, {k: v.to(DEV) for k, v in synth.synth_checkpoint(TINY, 3).items()}, device=DEV)


def _ids(name, *shape):
    return synth.token_ids(shape, V, 3, f"rules-state/{name}")


def _bits(words):
    return (words.cpu()[:, torch.arange(V) // 32].long() >> (torch.arange(V) % 32)) & 1


def _run(eng, rules, prefix, prompt, rep, full, steps=4):
    """A batch from its prompt on, checked step by step."""
    batch = prompt.shape[0]
    seen = torch.zeros(batch, V, dtype=torch.bool)
    seen[:, prefix] = True
    seen.scatter_(1, prompt, True)
    counts = torch.zeros(batch, V, dtype=torch.int64)
    token = (eng.prefill_full if full else eng.prefill)(prompt.to(DEV)).cpu()
    for step in range(steps):
        logits = eng.logits[:batch].float().cpu()
        x = torch.where(seen, torch.where(logits > 0, logits / torch.tensor(rep), logits * torch.tensor(rep)), logits)
        x = torch.where(counts > 0, x - 0.25 * counts, x)
        pick = torch.stack([(r == r.max()).nonzero()[0, 0] for r in x])
        assert torch.equal(token, pick), f"step {step}"
        counts.scatter_add_(1, pick[:, None], torch.ones_like(pick[:, None]))
        seen.scatter_(1, pick[:, None], True)
        assert torch.equal(rules.counts.cpu().long(), counts), f"step {step}"
        assert torch.equal(_bits(rules.seen).bool(), seen), f"step {step}"
        eng.decode_step()
        token = eng.current_ids.cpu()


@pytest.mark.parametrize("batch,backend,full", [(2, "cuda_core", False), (4, "tc", False), (3, "tc", True)])
@pytest.mark.parametrize("prefix_first", [False, True])
def test_batches_behind_one_prefix_and_another(runtime, batch, backend, full, prefix_first):
    """Two batches behind one prefix, with and without new rules for the second; then another prefix; then none of the
    old one's tokens left."""
    rules = TokenRules(batch, V, DEV)
    eng = DecodeEngine(runtime, batch, 64, linear_backend=backend, prefix_capacity=200, rules=rules)
    prefix = _ids("prefix", 200)

    def requests(rep):
        for b in range(batch):
            rules.set_request(b, repetition=rep, frequency=0.25)

    if prefix_first:
        eng.prefill_prefix(prefix)
        requests(1.5)
    else:
        requests(1.5)
        eng.prefill_prefix(prefix)
    _run(eng, rules, prefix, _ids("a", batch, 9), 1.5, full)
    eng.reset()
    requests(2.0)
    _run(eng, rules, prefix, _ids("b", batch, 5), 2.0, full)
    eng.reset()  # the same requests' rules again: nothing of the answers before
    _run(eng, rules, prefix, _ids("c", batch, 7), 2.0, full)
    eng.reset()
    other = _ids("other", 31)
    eng.prefill_prefix(other)
    _run(eng, rules, other, _ids("d", batch, 7), 2.0, full)
    eng.reset()
    requests(1.25)
    _run(eng, rules, other, _ids("e", batch, 4), 1.25, full)
    assert K.device_error() == 0


def test_no_prefix(runtime):
    rules = TokenRules(2, V, DEV)
    eng = DecodeEngine(runtime, 2, 64, rules=rules)
    none = torch.zeros(0, dtype=torch.int64)
    for name in ("n1", "n2"):
        for b in range(2):
            rules.set_request(b, repetition=1.5, frequency=0.25)
        _run(eng, rules, none, _ids(name, 2, 6), 1.5, False)
        eng.reset()


def test_tokens_noted_before_the_prefix_stay(runtime):
    rules = TokenRules(2, V, DEV)
    eng = DecodeEngine(runtime, 2, 64, prefix_capacity=8, rules=rules)
    extra = torch.tensor([[5, 40], [V - 1, -1]])
    rules.note_prompt(extra.to(DEV))
    eng.prefill_prefix(_ids("p", 8))
    want = torch.zeros(2, V, dtype=torch.bool)
    want[:, _ids("p", 8)] = True
    want[0, [5, 40]] = True
    want[1, V - 1] = True
    assert torch.equal(_bits(rules.seen).bool(), want)
