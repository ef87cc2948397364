"""A batch of different requests through the engine: shared prefix, adapters and token rules, alone and together.

The hidden rows are compared with the CPU oracle's fp32 mode (the adapters
merged into its fp32 weights, the prefix in front of every sequence's own
tokens) within the repository's bound of an engine step (``conftest.tol``); the
tokens are teacher-forced so that near-ties cannot make the runs diverge.  The
picks are checked on the engine's own logits, exactly.
"""

from __future__ import annotations

import dataclasses

import pytest
import torch

from conftest import tol
from leanstack_b200 import kernels as K
from leanstack_b200 import synth
from leanstack_b200.config import TINY
from leanstack_b200.engine import DecodeEngine
from leanstack_b200.leanserve import materialize_from_tensors
from leanstack_b200.requests import AdapterBank, TokenRules
from leanstack_b200.speculative import SpeculativeDecoder
from oracle import qwen_oracle as qo

pytestmark = pytest.mark.gpu
DEV = "cuda"
SEED = 3
TARGETS = {"qkv": "qkv_proj", "o": "o_proj", "gate_up": "gate_up_proj", "down": "down_proj"}


@pytest.fixture(scope="module")
def checkpoint():
    return synth.synth_checkpoint(TINY, SEED)


@pytest.fixture(scope="module")
def runtime(checkpoint):
    return materialize_from_tensors(TINY, {k: v.to(DEV) for k, v in checkpoint.items()}, device=DEV)


def _ids(name, *shape):
    return synth.token_ids(shape, TINY.vocab_size, SEED, f"requests/{name}")


def _bank(count=3, rank=16):
    """Adapters whose effect is as large as the linears' own (unit-variance activations through both)."""
    bank = AdapterBank(TINY, count, rank, DEV)
    g = torch.Generator().manual_seed(7)
    weights = []
    for i in range(count):
        w = {}
        for layer in range(TINY.num_hidden_layers):
            for t, (k, n) in bank.shapes.items():
                r = rank - 8 * (i % 2)  # every other one of a lower rank
                w[layer, t] = ((torch.randn(r, k, generator=g) * k ** -0.5).bfloat16(),
                               (torch.randn(n, r, generator=g) * 0.1).bfloat16())
        bank.load(i, w, 0.5 + 0.25 * i)
        weights.append((w, 0.5 + 0.25 * i))
    return bank, weights


def _oracle(checkpoint, weights=None, adapter=-1):
    """The fp32 oracle, an adapter merged into its weights."""
    m = qo.OracleModel.from_checkpoint(TINY, checkpoint, precision="fp32")
    if adapter < 0:
        return m
    w, s = weights[adapter]
    layers = []
    for i, layer in enumerate(m.layers):
        merged = {name: getattr(layer, name) + s * (w[i, t][1].float() @ w[i, t][0].float())
                  for t, name in TARGETS.items()}
        layers.append(dataclasses.replace(layer, **merged))
    return dataclasses.replace(m, layers=layers)


def _oracle_rows(prefix_model, model, prefix, own):
    """Final hidden row after each of ``own``'s tokens, the prefix's K/V made by ``prefix_model``."""
    kv = model.new_kv(1, 256)
    if len(prefix):
        qo.stack_forward(prefix_model, qo.embed(prefix_model, prefix[None]), kv, model.rope(256))
    return qo.stack_forward(model, qo.embed(model, own[None]), kv, model.rope(256))[0]


def _check_rows(eng, step, want):
    """The hidden rows of the engine's last head against the oracle's at own position ``step`` of each sequence."""
    got = eng.last_head_rows().float().cpu()
    ref = torch.stack([w[step] for w in want])
    assert (got - ref).abs().max().item() <= tol(ref), f"step {step}"


@pytest.mark.parametrize("batch,backend", [(1, "auto"), (3, "cuda_core"), (3, "tc"), (5, "auto")])
@pytest.mark.parametrize("full", [False, True])
def test_shared_prefix(checkpoint, runtime, batch, backend, full):
    prefix, prompt, forced = _ids("prefix", 83), _ids("prompt", batch, 9), _ids("forced", batch, 4)
    eng = DecodeEngine(runtime, batch, 64, linear_backend=backend, prefix_capacity=90)
    eng.prefill_prefix(prefix)
    model = _oracle(checkpoint)
    want = [_oracle_rows(model, model, prefix, torch.cat([prompt[b], forced[b]])) for b in range(batch)]
    (eng.prefill_full if full else eng.prefill)(prompt.to(DEV))
    _check_rows(eng, 8, want)
    for i in range(4):
        eng.set_next_ids(forced[:, i].to(DEV))
        eng.decode_step()  # the second and later ones replay a graph
        _check_rows(eng, 9 + i, want)
    assert K.device_error() == 0
    eng.reset()  # another prefix, another length: the captured step must not live on
    prefix2 = _ids("prefix2", 17)
    eng.prefill_prefix(prefix2)
    want = [_oracle_rows(model, model, prefix2, torch.cat([prompt[b], forced[b]])) for b in range(batch)]
    eng.prefill(prompt.to(DEV))
    eng.set_next_ids(forced[:, 0].to(DEV))
    eng.decode_step()
    _check_rows(eng, 9, want)
    assert K.device_error() == 0


@pytest.mark.parametrize("full", [False, True])
@pytest.mark.parametrize("ids,prefix_adapter", [([0], -1), ([0, -1, 2, 1, 2], -1), ([1, 1, 1], 1)])
def test_adapters_behind_a_prefix(checkpoint, runtime, ids, prefix_adapter, full):
    bank, weights = _bank()
    batch = len(ids)
    prefix, prompt, forced = _ids("aprefix", 40), _ids("aprompt", batch, 20), _ids("aforced", batch, 3)
    eng = DecodeEngine(runtime, batch, 64, prefix_capacity=40, adapters=bank)
    assert eng.backend == "tc"
    eng.set_adapters(ids)
    eng.prefill_prefix(prefix, adapter=prefix_adapter)
    base = _oracle(checkpoint, weights, prefix_adapter)
    models = {i: _oracle(checkpoint, weights, i) for i in set(ids)}
    want = [_oracle_rows(base, models[a], prefix, torch.cat([prompt[b], forced[b]])) for b, a in enumerate(ids)]
    plain = _oracle_rows(base, _oracle(checkpoint), prefix, torch.cat([prompt[0], forced[0]]))
    assert (want[0][-1] - plain[-1]).abs().max() > 4 * tol(plain[-1])  # the adapter matters
    (eng.prefill_full if full else eng.prefill)(prompt.to(DEV))
    _check_rows(eng, 19, want)
    for i in range(3):
        eng.set_next_ids(forced[:, i].to(DEV))
        eng.decode_step()
        _check_rows(eng, 20 + i, want)
    assert K.device_error() == 0


def test_adapters_change_under_a_captured_step(runtime):
    """Rewriting the adapter ids between replays equals eager steps with the same ids, bit for bit."""
    bank, _ = _bank()
    prompt = _ids("swap", 4, 12).to(DEV)
    rows = []
    for graph in (False, True):
        eng = DecodeEngine(runtime, 4, 64, use_graph=graph, adapters=bank)
        eng.set_adapters([0, 1, 2, -1])
        eng.prefill(prompt)
        out = []
        for ids in ([0, 1, 2, -1], [2, 2, -1, 0], [-1] * 4):
            eng.set_adapters(ids)
            eng.decode_step()
            out.append((eng.last_head_rows().clone(), eng.current_ids.clone()))
        rows.append(out)
    for (a, x), (b, y) in zip(*rows):
        assert torch.equal(a, b) and torch.equal(x, y)


def test_a_verify_pass_behind_a_prefix(checkpoint, runtime):
    """Every row of a verify pass (current and three proposals) against the oracle over prefix and own tokens; then
    whole speculative cycles run behind the prefix, also after it changes under their captured graph."""
    prefix, prompt, forced = _ids("vprefix", 50), _ids("vprompt", 2, 10), _ids("vforced", 2, 4)
    target = DecodeEngine(runtime, 2, 96, max_tokens_per_step=16, linear_backend="tc", prefix_capacity=60)
    target.prefill_prefix(prefix)
    target.prefill(prompt.to(DEV))
    model = _oracle(checkpoint)
    want = [_oracle_rows(model, model, prefix, torch.cat([prompt[b], forced[b]])) for b in range(2)]
    target.verify_inputs(3).copy_(forced.to(DEV))
    target.verify_step(3)
    got = target.last_head_rows().float().cpu().view(2, 4, -1)
    ref = torch.stack([w[10:] for w in want])
    assert (got - ref).abs().max().item() <= tol(ref)
    draft = DecodeEngine(runtime, 2, 96, max_tokens_per_step=16, linear_backend="tc", prefix_capacity=60)
    spec = SpeculativeDecoder(draft, target, 3, 8)
    runs = []
    for name in ("vprefix", "vprefix2", "vprefix"):
        for e in (draft, target):
            e.reset()
            e.prefill_prefix(_ids(name, 50 + 10 * (name == "vprefix2")))
        runs.append(spec.generate(prompt.to(DEV), 8))
        assert all(len(t) == 8 for t in runs[-1])
    assert runs[0] == runs[2] and runs[0] != runs[1]
    assert K.device_error() == 0


@pytest.mark.parametrize("batch,backend", [(2, "cuda_core"), (4, "tc")])
def test_token_rules(runtime, batch, backend):
    """Every pick follows the rules on the engine's own logits; the counts hold the answer, the seen bits prompt and answer."""
    V = TINY.vocab_size
    rules = TokenRules(batch, V, DEV, max_biases=3, grammar=True)
    eng = DecodeEngine(runtime, batch, 64, linear_backend=backend, rules=rules)
    for b in range(batch):
        rules.set_request(b, repetition=1.3, frequency=0.5, presence=1.0 + b, biases={5 + b: 2.0, 77: -float("inf")})
    g = torch.Generator().manual_seed(1)
    allowed = torch.rand(batch, V, generator=g) < 0.5
    words = (allowed.view(batch, -1, 32).long() << torch.arange(32)).sum(-1)
    rules.allowed.copy_(torch.where(words >= 2 ** 31, words - 2 ** 32, words).int())
    prompt = _ids("rprompt", batch, 11)
    seen = torch.zeros(batch, V, dtype=torch.bool).scatter_(1, prompt, True)
    counts = torch.zeros(batch, V, dtype=torch.int64)
    tokens = [eng.prefill(prompt.to(DEV)).cpu()]
    for step in range(8):
        logits = eng.logits[:batch].float().cpu()
        x = torch.where(seen, torch.where(logits > 0, logits / torch.tensor(1.3), logits * torch.tensor(1.3)), logits)
        pres = torch.arange(batch)[:, None] + 1.0
        x = torch.where(counts > 0, (x - 0.5 * counts) - pres, x)
        for b in range(batch):
            x[b, 5 + b] += 2.0
        x[:, 77] = float("-inf")
        x = x.masked_fill(~allowed, float("-inf"))
        pick = torch.stack([(r == r.max()).nonzero()[0, 0] for r in x])
        assert torch.equal(tokens[-1], pick), f"step {step}"
        counts.scatter_add_(1, pick[:, None], torch.ones_like(pick[:, None]))
        seen.scatter_(1, pick[:, None], True)
        assert torch.equal(rules.counts.cpu().long(), counts)
        eng.decode_step()
        tokens.append(eng.current_ids.cpu())
    assert K.device_error() == 0


def test_all_three_together(runtime):
    """Prefix, adapters and rules in one batch: captured steps equal eager ones bit for bit, tokens and state."""
    bank, _ = _bank()
    batch, V = 6, TINY.vocab_size
    prefix, prompt = _ids("tprefix", 130), _ids("tprompt", batch, 7).to(DEV)
    runs = []
    for graph in (False, True):
        rules = TokenRules(batch, V, DEV, max_biases=2, grammar=True)
        for b in range(batch):
            rules.set_request(b, repetition=1.1, frequency=0.2, presence=0.5, biases={b: 1.0})
        rules.allowed[2].fill_(0)
        rules.allowed[2, 3:5].fill_(-1)  # this request may say 64 tokens only
        eng = DecodeEngine(runtime, batch, 64, use_graph=graph, prefix_capacity=130, adapters=bank, rules=rules)
        eng.set_adapters([0, 1, -1, 2, 0, 0])
        eng.prefill_prefix(prefix)
        out = [eng.prefill(prompt)]
        for _ in range(10):
            eng.decode_step()
            out.append(eng.current_ids.clone())
        assert K.device_error() == 0
        runs.append((torch.stack(out, 1), rules.counts.clone(), rules.seen.clone(), eng.kv.key_cache.clone()))
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    tokens = runs[0][0]
    assert ((tokens[2] >= 96) & (tokens[2] < 160)).all()
    assert torch.equal(runs[0][1].sum(1).cpu(), torch.full((batch,), 11))


def test_the_plain_engine_is_unchanged_by_room_for_a_prefix(runtime):
    """An engine with an unused prefix arena gives the plain engine's bits."""
    prompt = _ids("uprompt", 3, 9).to(DEV)
    outs = []
    for cap in (0, 32):
        eng = DecodeEngine(runtime, 3, 64, prefix_capacity=cap)
        toks = eng.generate(prompt, 6)
        outs.append((toks, eng.last_head_rows().clone(), eng.kernel_launches_per_step()))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1]) and outs[0][2] == outs[1][2]


def test_refusals(runtime):
    bank, _ = _bank(2, 8)
    eng = DecodeEngine(runtime, 2, 32)
    with pytest.raises(ValueError, match="no room for a prefix"):
        eng.prefill_prefix(_ids("r", 4))
    with pytest.raises(ValueError, match="no adapter bank"):
        eng.set_adapters([0, 0])
    eng = DecodeEngine(runtime, 2, 32, prefix_capacity=8, adapters=bank)
    with pytest.raises(ValueError, match="1 <= P <= 8"):
        eng.prefill_prefix(_ids("r", 9))
    with pytest.raises(ValueError, match="no adapter 2"):
        eng.prefill_prefix(_ids("r", 4), adapter=2)
    with pytest.raises(ValueError, match="adapter ids below 2"):
        eng.set_adapters([0, 2])
    eng.prefill(_ids("r2", 2, 3))
    with pytest.raises(ValueError, match="already hold tokens"):
        eng.prefill_prefix(_ids("r", 4))
    with pytest.raises(ValueError, match="split partials"):
        DecodeEngine(runtime, 1, 32, linear_backend="cuda_core", adapters=bank)
    rules = TokenRules(2, TINY.vocab_size, DEV)
    with pytest.raises(ValueError, match="token rules for 2 rows"):
        DecodeEngine(runtime, 3, 32, rules=rules)
    ruled = DecodeEngine(runtime, 2, 32, max_tokens_per_step=8, rules=rules)
    with pytest.raises(ValueError, match="no token rules"):
        ruled.verify_step(1)
    with pytest.raises(ValueError, match="no token rules"):
        SpeculativeDecoder(ruled, ruled, 1, 4)
    with pytest.raises(ValueError, match="room for 0"):
        rules.set_request(0, biases={1: 1.0})
    with pytest.raises(ValueError, match="repetition must be positive"):
        rules.set_request(0, repetition=0.0)
    with pytest.raises(ValueError, match="multiple of 8"):
        AdapterBank(TINY, 1, 12, DEV)
    with pytest.raises(ValueError, match="do not fit"):
        bank.load(0, {(0, "o"): (torch.zeros(16, 512), torch.zeros(512, 16))}, 1.0)
