"""A request whose rules allow no token picks -1 and goes on as padding: no error, and the other rows' tokens as without
it, in eager and captured steps; once its rules allow a token again it picks one."""

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


def _run(runtime, batch, backend, graph, prefix, banned):
    """Tokens [batch, 10]; row `banned` may say nothing from step 3 to 6 and in the very first pick."""
    rules = TokenRules(batch, V, DEV, grammar=True)
    eng = DecodeEngine(runtime, batch, 64, linear_backend=backend, use_graph=graph, rules=rules,
                       prefix_capacity=20 if prefix else 0)
    K.device_error(clear=True)
    for b in range(batch):
        rules.set_request(b, repetition=1.2, presence=0.5)
    if prefix:
        eng.prefill_prefix(synth.token_ids((20,), V, 3, "none/prefix"))
    out = []
    for step in range(10):
        if banned is not None:
            rules.allowed[banned].fill_(0 if step == 0 or 3 <= step <= 6 else -1)
        if step == 0:
            out.append(eng.prefill(synth.token_ids((batch, 6), V, 3, "none/prompt").to(DEV)))
        else:
            eng.decode_step()
            out.append(eng.current_ids.clone())
        assert K.device_error() == 0, f"step {step}"
        assert torch.isfinite(eng.last_head_rows().float()).all()
    return torch.stack(out, 1), rules


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("batch,backend", [(1, "cuda_core"), (3, "cuda_core"), (4, "tc")])
def test_a_row_without_a_token(runtime, batch, backend, prefix):
    banned = batch // 2
    others = [b for b in range(batch) if b != banned]
    want, _ = _run(runtime, batch, backend, False, prefix, None)
    for graph in (False, True):
        got, rules = _run(runtime, batch, backend, graph, prefix, banned)
        assert torch.equal(got[others], want[others])
        none = torch.zeros(10, dtype=torch.bool, device=DEV)
        none[[0, 3, 4, 5, 6]] = True
        assert torch.equal(got[banned] == -1, none) and (got >= -1).all() and (got < V).all()
        assert rules.counts[banned].sum().item() == 5  # a pick of nothing is not counted
