"""Penalties, biases and grammar masks on logits, and the greedy pick under them.

The processed logits are compared with the rules in 64 bits: at most seven fp32
roundings of values no larger than S = |l| max(rep, 1 / rep) + frequency count
+ presence + sum |bias| (plus one more per further bias of a token), so they
stay within (8 + biases) x 2^-24 x S.  The picked id must hold the largest
processed logit of the kernel's own output at its lowest index, and its 64-bit
value must be within the same bound of the 64-bit maximum.
"""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pack(bits):
    b, v = bits.shape
    words = (v + 31) // 32
    full = torch.zeros(b, words * 32, dtype=torch.int64, device=bits.device)
    full[:, :v] = bits
    w = (full.view(b, words, 32) << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


def _state(m, vocab, dtype, allowed, history, biases, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    st = {"logits": (torch.randn(m, vocab, generator=g, device=DEV) * 3).to(dtype)}
    tokens = (torch.rand(m, history, generator=g, device=DEV) ** 2 * vocab).long()
    st["counts"] = torch.zeros(m, vocab, device=DEV, dtype=torch.int32)
    answer = tokens[:, history // 2:]
    st["counts"].scatter_add_(1, answer, torch.ones_like(answer, dtype=torch.int32))
    st["seen_bits"] = torch.zeros(m, vocab, device=DEV, dtype=torch.bool).scatter_(1, tokens, True)
    st["repetition"] = torch.rand(m, generator=g, device=DEV) * 0.6 + 0.9
    st["frequency"] = torch.rand(m, generator=g, device=DEV) - 0.2
    st["presence"] = torch.rand(m, generator=g, device=DEV) * 2 - 0.5
    if biases:
        st["bias_ids"] = (torch.rand(m, biases, generator=g, device=DEV) * (vocab + 2)).int() - 1  # some outside
        st["bias_ids"][:, 0] = st["bias_ids"][:, biases // 2]  # the same token twice
        st["bias_values"] = torch.randn(m, biases, generator=g, device=DEV) * 5
    if allowed is not None:
        st["allowed_bits"] = torch.rand(m, vocab, generator=g, device=DEV) < allowed
    return st


def _rules(st):
    """(processed logits in float64 with -inf where banned, S)."""
    x = st["logits"].double()
    m, vocab = x.shape
    rep, freq, pres = (st[k].double()[:, None] for k in ("repetition", "frequency", "presence"))
    n = st["counts"].double()
    s = x.abs() * torch.maximum(rep, 1 / rep) + (freq * n).abs() + pres.abs()
    x = torch.where(st["seen_bits"], torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(n > 0, x - freq * n - pres, x)
    if "bias_ids" in st:
        ids = st["bias_ids"].long()
        inside = (ids >= 0) & (ids < vocab)
        vals = torch.where(inside, st["bias_values"].double(), 0.0)
        x = x + torch.zeros_like(x).scatter_add_(1, ids.clamp(0, vocab - 1), vals)
        s = s + torch.zeros_like(x).scatter_add_(1, ids.clamp(0, vocab - 1), vals.abs())
    if "allowed_bits" in st:
        x = x.masked_fill(~st["allowed_bits"], float("-inf"))
    return x, s


def _call(st, **kw):
    return K.constrained_argmax(st["logits"], counts=st["counts"], seen=pack(st["seen_bits"]),
                                repetition=st["repetition"], frequency=st["frequency"], presence=st["presence"],
                                bias_ids=st.get("bias_ids"), bias_values=st.get("bias_values"),
                                allowed=pack(st["allowed_bits"]) if "allowed_bits" in st else None, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 7, 31, 32, 33, 64, 1000, 4096, 32001, 151936])
@pytest.mark.parametrize("m,allowed,biases", [(1, None, 0), (3, 0.9, 5), (5, 0.01, 40), (36, None, 2)])
def test_processed_logits_and_pick(dtype, vocab, m, allowed, biases):
    st = _state(m, vocab, dtype, allowed, 50, biases)
    out = torch.full((m, vocab), float("nan"), device=DEV)
    ids = _call(st, out_logits=out)
    want, s = _rules(st)
    banned = want == float("-inf")
    assert torch.equal(out == float("-inf"), banned)
    err = (out.double() - want).masked_fill(banned, 0.0).abs()
    bound = (8 + biases) * 2 ** -24 * s
    assert (err <= bound).all()
    for r in range(m):
        if banned[r].all():
            assert int(ids[r]) == -1
            continue
        assert int(ids[r]) == int((out[r] == out[r].max()).nonzero()[0])
        i = int(ids[r])
        assert want[r, i].item() >= want[r].max().item() - 2 * bound[r].max().item()
    assert torch.equal(_call(st), ids)  # without the written logits


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,vocab", [(1, 1 << 20), (20, 1 << 20), (33, 700001), (300, 9999)])
def test_large_vocabularies_and_many_rows(dtype, m, vocab):
    st = _state(m, vocab, dtype, 0.5, 40, 3)
    want, s = _rules(st)
    ids = _call(st)
    at = want.gather(1, ids[:, None])[:, 0]
    assert (at >= want.amax(1) - 2 * 11 * 2 ** -24 * s.amax(1)).all()


def test_plain_argmax_without_rules():
    """No rules at all: torch.argmax of the row, lowest index on ties (bf16 rows hold many)."""
    g = torch.Generator(device=DEV).manual_seed(4)
    logits = torch.randn(6, 5001, generator=g, device=DEV).mul_(8).round_().bfloat16()
    want = torch.stack([(r == r.max()).nonzero()[0, 0] for r in logits.float()])
    assert torch.equal(K.constrained_argmax(logits), want)
    assert torch.equal(K.constrained_argmax(logits.float()), want)


def test_infinities_and_nan():
    inf, nan = float("inf"), float("nan")
    rows = torch.tensor([
        [nan, 1.0, 2.0, nan],  # NaN is never picked
        [nan, nan, nan, nan],  # nothing to pick
        [-inf, -inf, -inf, -inf],  # candidates all the same: the lowest
        [inf, 3.0, inf, 1.0],
        [5.0, inf, nan, 4.0],  # the banned places hold the largest and the NaN
        [-3e38, -3.3e38, 9.0, 0.0],
    ], device=DEV)
    allowed = torch.ones(6, 4, dtype=torch.bool, device=DEV)
    allowed[4, 1] = allowed[4, 2] = False
    allowed[2, 0] = False
    allowed[5, 2:] = False
    for dtype in (torch.float32, torch.bfloat16):
        ids = K.constrained_argmax(rows.to(dtype), allowed=pack(allowed))
        assert ids.tolist() == [2, -1, 1, 0, 0, 0]
    none = K.constrained_argmax(rows, allowed=torch.zeros(6, 1, device=DEV, dtype=torch.int32))
    assert none.tolist() == [-1] * 6


def test_a_far_minus_infinity_behind_nan():
    """Whole groups of NaN before the only candidates, which are -inf: the lowest of those is picked."""
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.full((3, 9000), float("nan"), device=DEV, dtype=dtype)
        logits[0, 8500] = logits[0, 8999] = float("-inf")
        logits[1, 17] = float("-inf")
        logits[1, 4000] = -2.0
        assert K.constrained_argmax(logits).tolist() == [8500, 4000, -1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [40, 9000, 9003])
def test_rows_without_a_finite_candidate(dtype, vocab):
    """Only -inf left: the lowest token that is allowed and -inf, biased or not; a biased one above -inf wins."""
    inf, nan = float("inf"), float("nan")
    m = 8
    logits = torch.full((m, vocab), nan, device=DEV, dtype=dtype)
    allowed = torch.ones(m, vocab, dtype=torch.bool, device=DEV)
    ids = torch.full((m, 2), -1, device=DEV, dtype=torch.int32)
    vals = torch.zeros(m, 2, device=DEV)
    want = []
    logits[0, vocab - 2] = -inf  # behind NaN
    want.append(vocab - 2)
    logits[1] = -inf  # the lowest is banned
    allowed[1, :7] = False
    want.append(7)
    logits[2] = 5.0  # nothing allowed
    allowed[2] = False
    want.append(-1)
    logits[3] = 1.0  # biased to -inf, the only one allowed
    allowed[3] = False
    allowed[3, 33] = True
    ids[3, 0], vals[3, 0] = 33, -inf
    want.append(33)
    logits[4] = -inf  # the lowest one is biased, which leaves it -inf
    ids[4, 0], vals[4, 0] = 0, 3.0
    want.append(0)
    logits[5] = -inf  # one of them is forced above
    ids[5, 1], vals[5, 1] = 38, inf  # -inf + inf: NaN, no candidate
    ids[5, 0], vals[5, 0] = 0, inf
    want.append(1)
    logits[6] = -inf
    logits[6, 20] = -3.0  # finite, but biased away
    ids[6, 0], vals[6, 0] = 20, -inf
    want.append(0)
    logits[7] = 2.0  # every token of the largest group but one is biased down
    logits[7, 8:16] = 4.0
    ids7 = torch.tensor([8, 9], device=DEV, dtype=torch.int32)
    ids[7], vals[7] = ids7, torch.tensor([-1.0, -3.0], device=DEV)
    want.append(10)
    out = torch.empty(m, vocab, device=DEV)
    got = K.constrained_argmax(logits, allowed=pack(allowed), bias_ids=ids, bias_values=vals, out_logits=out)
    assert got.tolist() == want
    ref = logits.float()
    for r in range(m):
        for k in range(2):
            if ids[r, k] >= 0:
                ref[r, ids[r, k].item()] += vals[r, k]
    ref[~allowed] = -inf
    assert torch.equal(torch.nan_to_num(out, nan=7e4), torch.nan_to_num(ref, nan=7e4))


@pytest.mark.parametrize("cap", [1, 127, 128, 129, 512, 513, 1100])
@pytest.mark.parametrize("vocab", [700, 5003])
def test_long_bias_lists(cap, vocab):
    """Lists longer than a stage and than the pick's threads, with repeated tokens far apart."""
    g = torch.Generator(device=DEV).manual_seed(cap)
    m = 3
    logits = torch.randn(m, vocab, generator=g, device=DEV)
    ids = torch.randint(-3, vocab + 3, (m, cap), generator=g, device=DEV, dtype=torch.int32)
    if cap > 2:
        ids[:, cap - 1] = ids[:, 0]
        ids[1] = 5  # one token only
    vals = torch.randint(-8, 9, (m, cap), generator=g, device=DEV).float() / 4  # (sums of quarters: exact)
    out = torch.empty(m, vocab, device=DEV)
    got = K.constrained_argmax(logits, bias_ids=ids, bias_values=vals, out_logits=out)
    steps = torch.zeros(m, vocab, device=DEV)
    inside = (ids >= 0) & (ids < vocab)
    steps.scatter_add_(1, ids.clamp(0, vocab - 1).long(), vals * inside)
    want = logits + steps
    assert torch.equal(out, want)
    assert torch.equal(got, torch.stack([(r == r.max()).nonzero()[0, 0] for r in want]))


def test_a_bias_of_minus_infinity_bans_and_plus_infinity_forces():
    logits = torch.arange(100, device=DEV, dtype=torch.float32).expand(2, 100).contiguous()
    ids = torch.tensor([[99, 98], [3, 99]], device=DEV, dtype=torch.int32)
    vals = torch.tensor([[float("-inf"), float("-inf")], [float("inf"), 1.0]], device=DEV)
    assert K.constrained_argmax(logits, bias_ids=ids, bias_values=vals).tolist() == [97, 3]


@pytest.mark.parametrize("vocab", [40, 50263])
def test_record_counts_the_pick(vocab):
    """Repeated picks move the counts; a strong presence penalty makes every pick a new token."""
    m = 4
    st = _state(m, vocab, torch.bfloat16, None, 10, 0)
    st["frequency"].zero_()
    st["presence"].fill_(1000.0)
    st["repetition"].fill_(1.0)
    seen = pack(st["seen_bits"])
    before = st["counts"].clone()
    picks = []
    for _ in range(6):
        picks.append(K.constrained_argmax(st["logits"], counts=st["counts"], seen=seen, repetition=st["repetition"],
                                          frequency=st["frequency"], presence=st["presence"], record=True))
    picks = torch.stack(picks, 1)
    for r in range(m):
        assert len(set(picks[r].tolist())) == 6
    assert torch.equal(st["counts"], before.scatter_add_(1, picks, torch.ones_like(picks, dtype=torch.int32)))
    assert torch.equal(seen, pack(st["seen_bits"].scatter_(1, picks, True)))
    # a row with nothing allowed records nothing
    counts, words = st["counts"].clone(), seen.clone()
    ids = K.constrained_argmax(st["logits"], counts=st["counts"], seen=seen, allowed=torch.zeros_like(seen), record=True)
    assert ids.tolist() == [-1] * m and torch.equal(st["counts"], counts) and torch.equal(seen, words)


def test_token_stats_add():
    vocab, batch = 1000, 3
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, vocab, (batch, 700), generator=g)
    ids[0, 100:] = -1  # padding
    ids[1, :] = 31  # the same token again and again
    want = torch.zeros(batch, vocab, dtype=torch.int64)
    for b in range(batch):
        want[b] = torch.bincount(ids[b][ids[b] >= 0], minlength=vocab)
    seen = torch.zeros(batch, 32, device=DEV, dtype=torch.int32)
    counts = torch.zeros(batch, vocab, device=DEV, dtype=torch.int32)
    K.token_stats_add(ids.to(DEV), seen, vocab)
    assert torch.equal(seen.cpu(), pack(want > 0))
    K.token_stats_add(ids.to(DEV), seen, vocab, counts=counts)
    assert torch.equal(counts.cpu().long(), want) and torch.equal(seen.cpu(), pack(want > 0))
    K.token_stats_add(torch.empty(batch, 0, device=DEV, dtype=torch.int64), seen, vocab)
    K.device_error(clear=True)
    K.token_stats_add(torch.tensor([[vocab], [2 ** 40], [5]], device=DEV), seen, vocab, counts=counts)
    assert K.device_error(clear=True) == 1  # LS_ERR_INVALID_ARGUMENT
    want[2, 5] += 1
    assert torch.equal(counts.cpu().long(), want)


def test_replay_follows_the_state():
    """One captured pick replayed on its own recorded state equals the same picks made one by one."""
    st = _state(2, 5000, torch.bfloat16, 0.5, 30, 3)
    seen = pack(st["seen_bits"])
    allowed = pack(st["allowed_bits"])
    kw = {k: st[k] for k in ("repetition", "frequency", "presence", "bias_ids", "bias_values")}
    c1, s1, c2, s2 = st["counts"].clone(), seen.clone(), st["counts"].clone(), seen.clone()
    want = [K.constrained_argmax(st["logits"], counts=c1, seen=s1, allowed=allowed, record=True, **kw).clone()
            for _ in range(5)]
    out = torch.empty(2, device=DEV, dtype=torch.int64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.constrained_argmax(st["logits"], counts=c2, seen=s2, allowed=allowed, record=True, out_ids=out, **kw)
    for w in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    assert torch.equal(c1, c2) and torch.equal(s1, s2)


def test_refusals():
    st = _state(2, 100, torch.bfloat16, None, 5, 2)
    seen = pack(st["seen_bits"])
    with pytest.raises(K.nat.LeanB200Error, match="come together"):
        K.constrained_argmax(st["logits"], counts=st["counts"])
    with pytest.raises(K.nat.LeanB200Error, match="need counts and seen"):
        K.constrained_argmax(st["logits"], presence=st["presence"])
    with pytest.raises(K.nat.LeanB200Error, match="need counts and seen"):
        K.constrained_argmax(st["logits"], record=True)
    with pytest.raises(ValueError, match="come together"):
        K.constrained_argmax(st["logits"], bias_ids=st["bias_ids"])
    with pytest.raises(ValueError, match="allowed must have shape"):
        K.constrained_argmax(st["logits"], allowed=seen[:, :3].contiguous())
    with pytest.raises(TypeError, match="bf16 or fp32"):
        K.constrained_argmax(st["logits"].half())
    with pytest.raises(TypeError, match="repetition"):
        K.constrained_argmax(st["logits"], counts=st["counts"], seen=seen, repetition=st["repetition"].double())
    with pytest.raises(ValueError, match="contiguous"):
        K.constrained_argmax(st["logits"].t().contiguous().t())
    with pytest.raises(TypeError, match="ids"):
        K.token_stats_add(torch.zeros(2, 3, device=DEV, dtype=torch.int32), seen, 100)
