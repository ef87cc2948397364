"""The multi-request operators at once on several streams, and where offsets pass 32 bits."""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _prefix_case(batch, q_len, prefix, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF16)  # noqa: E731
    hq, hkv, slots = 16, 4, 200 + q_len
    args = (r(batch * q_len, hq * 128), r(hkv, prefix, 128), r(hkv, prefix, 128), r(batch, hkv, slots, 128),
            r(batch, hkv, slots, 128), batch, q_len, hq, hkv, 128, prefix, slots, 0.088)
    pos = (torch.arange(batch, device=DEV, dtype=torch.int32) * 17) % 200
    return lambda: K.shared_prefix_attention(*args, cache_pos=pos)


def _lora_case(batch, q_len, rank, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(batch * q_len, 1024, generator=g, device=DEV).to(BF16)
    a = torch.randn(5, rank, 1024, generator=g, device=DEV).to(BF16)
    b = torch.randn(5, 2048, rank, generator=g, device=DEV).to(BF16)
    s = torch.rand(5, generator=g, device=DEV)
    ids = torch.arange(batch, device=DEV, dtype=torch.int32) % 6 - 1
    return lambda: K.lora_delta(x, a, b, s, ids, q_len)


def _rules_case(m, vocab, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = torch.randn(m, vocab, generator=g, device=DEV).to(BF16)
    seen = torch.randint(-2 ** 31, 2 ** 31, (m, (vocab + 31) // 32), generator=g, device=DEV).int()
    counts = torch.ones(m, vocab, device=DEV, dtype=torch.int32)
    rep = torch.full((m,), 1.2, device=DEV)
    ids = torch.randint(0, vocab, (m, 30), generator=g, device=DEV, dtype=torch.int32)
    vals = torch.randn(m, 30, generator=g, device=DEV)

    def run():
        out = torch.empty(m, vocab, device=DEV)
        picked = K.constrained_argmax(logits, counts=counts, seen=seen, repetition=rep, bias_ids=ids, bias_values=vals,
                                      out_logits=out)
        return torch.cat([picked.float(), out.flatten()])

    return run


@pytest.mark.parametrize("make", [
    lambda s: _prefix_case(12, 1, 3001, s),  # key mode: strips beside the prefix
    lambda s: _prefix_case(2, 2, 700, s),  # few rows
    lambda s: _prefix_case(60, 3, 1500, s),  # row mode
    lambda s: _prefix_case(12, 80, 400, s),  # prompts
    lambda s: _lora_case(20, 1, 16, s),
    lambda s: _lora_case(6, 3, 72, s),
    lambda s: _lora_case(3, 100, 32, s),
    lambda s: _rules_case(3, 32000, s),
    lambda s: _rules_case(70, 50263, s),
], ids=["keys", "few", "rows", "full", "lora1", "lora2", "lora_prompt", "rules_few", "rules_many"])
def test_calls_at_once_on_three_streams(make):
    """Each call on its own operands and workspace: equal bits, whatever runs beside it."""
    cases = [make(seed) for seed in (1, 2, 3)]
    K.device_error(clear=True)
    want = [c() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(12):
        for i, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                got[i].append(c())
    torch.cuda.synchronize()
    assert K.device_error(clear=True) == 0
    for w, outs in zip(want, got):
        for o in outs:
            assert torch.equal(o, w)


def test_two_graphs_share_a_workspace():
    """Captured calls of different sizes on one workspace, replayed in turn."""
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF16)  # noqa: E731
    pos = torch.tensor([3, 60, 0], device=DEV, dtype=torch.int32)
    attn = (r(3, 2048), r(4, 900, 128), r(4, 900, 128), r(3, 4, 64, 128), r(3, 4, 64, 128), 3, 1, 16, 4, 128, 900, 64, 0.1)
    x, a, b = r(40, 512), r(3, 72, 512), r(3, 1024, 72)
    s, ids = torch.rand(3, device=DEV), torch.arange(40, device=DEV, dtype=torch.int32) % 3
    logits = r(9, 40000)
    calls = [lambda: K.shared_prefix_attention(*attn, cache_pos=pos, workspace=ws),
             lambda: K.lora_delta(x, a, b, s, ids, workspace=ws),
             lambda: K.constrained_argmax(logits, workspace=ws)]
    want = [c() for c in calls]
    graphs, outs = [], []
    for c in calls:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(c())
        graphs.append(gr)
    for order in ((0, 1, 2), (2, 0, 1), (1, 1, 0), (2, 2, 2)):
        for o in outs:
            o.zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in set(order):
            assert torch.equal(outs[i], want[i]), (order, i)


def test_caches_past_32_bits():
    """Own strips whose last offsets pass 2^32 bytes and 2^31 elements; the same rows in a small cache give the same bits."""
    batch, hq, hkv, big, prefix = 36, 8, 4, 131072, 300
    g = torch.Generator(device=DEV).manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF16)  # noqa: E731
    q, kp, vp, k, v = r(batch, hq * 128), r(hkv, prefix, 128), r(hkv, prefix, 128), r(batch, hkv, 64, 128), r(batch, hkv, 64, 128)
    pos = torch.arange(batch, device=DEV, dtype=torch.int32)
    kc = torch.empty(batch, hkv, big, 128, device=DEV, dtype=BF16)
    vc = torch.empty_like(kc)
    assert kc.numel() > 2 ** 31
    kc[:, :, :64] = k
    vc[:, :, :64] = v

    def run(kc, vc, slots, n=batch, workspace=None):
        return K.shared_prefix_attention(q[:n].contiguous(), kp, vp, kc, vc, n, 1, hq, hkv, 128, prefix, slots, 0.09,
                                         cache_pos=pos[:n].contiguous())

    want = run(k, v, 64).float()
    got = run(kc, vc, big).float()
    # the chunks of a strip depend on its room: equal up to their joins' fp32 roundings and one bf16 step
    assert ((got - want).abs() <= want.abs() * 2 ** -7 + 2 ** -9).all()


def test_adapters_past_32_bits():
    adapters, rank, k, n = 1800, 64, 64, 19456
    a = torch.empty(adapters, rank, k, device=DEV, dtype=BF16)
    b = torch.empty(adapters, n, rank, device=DEV, dtype=BF16)
    assert b.numel() > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(6)
    s = torch.ones(adapters, device=DEV)
    ids = torch.tensor([adapters - 1, 0, -1, adapters - 2], device=DEV, dtype=torch.int32)
    for i in (0, adapters - 2, adapters - 1):
        a[i] = torch.randn(rank, k, generator=g, device=DEV).to(BF16)
        b[i] = torch.randn(n, rank, generator=g, device=DEV).to(BF16)
    x = torch.randn(4, k, generator=g, device=DEV).to(BF16)
    small = torch.tensor([2, 0, -1, 1], device=DEV, dtype=torch.int32)
    pick = [0, adapters - 2, adapters - 1]
    want = K.lora_delta(x, a[pick].contiguous(), b[pick].contiguous(), s[:3].contiguous(), small)
    assert torch.equal(K.lora_delta(x, a, b, s, ids), want)
    for q_len in (4, 20):  # one sequence of a short length, prompts
        xs = torch.randn(3 * q_len, k, generator=g, device=DEV).to(BF16)
        want = K.lora_delta(xs, a[pick].contiguous(), b[pick].contiguous(), s[:3].contiguous(), small[:3].contiguous(), q_len)
        assert torch.equal(K.lora_delta(xs, a, b, s, ids[:3].contiguous(), q_len), want)


@pytest.mark.parametrize("vocab", [1 << 20, (1 << 20) - 3])
def test_rows_past_32_bits(vocab):
    m = 2060
    logits = torch.zeros(m, vocab, device=DEV, dtype=BF16)
    assert logits.numel() > 2 ** 31
    counts = torch.zeros(m, vocab, device=DEV, dtype=torch.int32)
    seen = torch.zeros(m, (vocab + 31) // 32, device=DEV, dtype=torch.int32)
    want = torch.arange(m, device=DEV) * 509 % vocab
    want[-1] = vocab - 1
    logits.scatter_(1, want[:, None], 5.0)
    got = K.constrained_argmax(logits, counts=counts, seen=seen, record=True)
    assert torch.equal(got, want)
    assert torch.equal(counts.argmax(1), want) and counts.sum().item() == m
    # a penalty of the recorded pick makes the next one the lowest other token
    got = K.constrained_argmax(logits, counts=counts, seen=seen, presence=torch.full((m,), 9.0, device=DEV))
    assert torch.equal(got, (want == 0).long())
