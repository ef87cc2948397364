"""The C++ front end and the Python checks behind it enqueue the same call: equal bits, the same errors."""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import _native as nat
from leanstack_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


class _Declines:
    """A front end that takes no call."""

    def __getattr__(self, name):
        return lambda *args: None


def _both(monkeypatch, fn):
    """fn's output by the front end and by the Python path; each must have gone its own way."""
    taken = []
    real = nat.front()

    class Spy:
        def __getattr__(self, name):
            def call(*args):
                done = getattr(real, name)(*args)
                taken.append(done is not None)
                return done
            return call

    monkeypatch.setattr(nat, "_FRONT", Spy())
    a = fn()
    monkeypatch.setattr(nat, "_FRONT", _Declines())
    b = fn()
    monkeypatch.setattr(nat, "_FRONT", real)
    assert taken == [True]
    return a, b


def _prefix(batch=3, q_len=1, prefix=50, slots=16):
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV, BF16)  # noqa: E731
    lens = torch.arange(batch, dtype=torch.int32, device=DEV)
    return [r(batch * q_len, 8 * 128), r(2, 64, 128), r(2, 64, 128), r(batch, 2, slots, 128), r(batch, 2, slots, 128),
            batch, q_len, 8, 2, 128, prefix, slots, 0.088], lens


def _lora():
    g = torch.Generator().manual_seed(3)
    return [torch.randn(4, 64, generator=g).to(DEV, BF16), torch.randn(2, 8, 64, generator=g).to(DEV, BF16),
            torch.randn(2, 32, 8, generator=g).to(DEV, BF16), torch.tensor([1.0, 0.5], device=DEV),
            torch.tensor([0, 1, -1, 1], dtype=torch.int32, device=DEV)]


@pytest.mark.parametrize("workspace", [False, True])
@pytest.mark.parametrize("cursor", [False, True])
def test_shared_prefix_attention(monkeypatch, cursor, workspace):
    args, lens = _prefix()
    kw = {"cache_pos": lens} if cursor else {"uniform_past": 3}

    def run():
        extra = dict(kw)
        if workspace:
            extra["workspace"] = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
            extra["out"] = torch.empty(3, 8 * 128, dtype=BF16, device=DEV)
        got = K.shared_prefix_attention(*args, **extra)
        assert not workspace or got is extra["out"]
        return got

    a, b = _both(monkeypatch, run)
    assert torch.equal(a, b) and a.shape == (3, 8 * 128)


@pytest.mark.parametrize("accumulate", [False, True])
def test_lora_delta(monkeypatch, accumulate):
    args = _lora()
    a, b = _both(monkeypatch, lambda: K.lora_delta(*args, accumulate=accumulate,
                                                   out=torch.ones(4, 32, device=DEV) if accumulate else None))
    assert torch.equal(a, b) and a.dtype == torch.float32


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("biases", [None, 0, 3])
def test_constrained_argmax(monkeypatch, dtype, biases):
    g = torch.Generator().manual_seed(4)
    m, vocab = 3, 1000
    logits = torch.randn(m, vocab, generator=g).to(DEV, dtype)
    kw = {}
    if biases is not None:
        kw["bias_ids"] = torch.full((m, biases), 7, dtype=torch.int32, device=DEV)
        kw["bias_values"] = torch.full((m, biases), 9.0, device=DEV)
    states = []

    def run():
        st = dict(counts=torch.zeros(m, vocab, dtype=torch.int32, device=DEV),
                  seen=torch.full((m, 32), 0x0F0F0F0F, dtype=torch.int32, device=DEV),
                  repetition=torch.full((m,), 1.3, device=DEV), frequency=torch.full((m,), 0.1, device=DEV),
                  presence=torch.full((m,), 0.2, device=DEV),
                  allowed=torch.full((m, 32), -1, dtype=torch.int32, device=DEV),
                  out_logits=torch.empty(m, vocab, device=DEV))
        states.append(st)
        return K.constrained_argmax(logits, record=True, **st, **kw)

    a, b = _both(monkeypatch, run)
    assert torch.equal(a, b)
    for name in ("counts", "seen", "out_logits"):
        assert torch.equal(states[0][name], states[1][name]), name
    assert states[0]["counts"].sum().item() == m


def test_another_stream_and_a_captured_call():
    args, lens = _prefix()
    want = K.shared_prefix_attention(*args, cache_pos=lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = K.shared_prefix_attention(*args, cache_pos=lens)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = K.shared_prefix_attention(*args, cache_pos=lens)
        delta = K.lora_delta(*_LORA)
        ids = K.constrained_argmax(delta)
    for _ in range(3):
        got.zero_()
        ids.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert torch.equal(ids, K.constrained_argmax(K.lora_delta(*_LORA)))


_LORA = None


@pytest.fixture(autouse=True)
def _operands():
    global _LORA
    _LORA = _lora()


def test_operands_that_the_python_path_names():
    args, lens = _prefix()
    for i, bad in ((0, args[0].float()), (1, args[1].transpose(0, 1)), (3, args[3][:2]), (4, args[4].cpu())):
        wrong = list(args)
        wrong[i] = bad
        with pytest.raises((TypeError, ValueError)):
            K.shared_prefix_attention(*wrong, cache_pos=lens)
    with pytest.raises(ValueError, match="cache_pos"):
        K.shared_prefix_attention(*args, cache_pos=lens[:2])
    with pytest.raises(nat.LeanB200Error, match="LS_ERR_KV_OVERFLOW"):
        K.shared_prefix_attention(*args, uniform_past=16)
    with pytest.raises(nat.LeanB200Error, match="LS_ERR_WORKSPACE"):
        K.shared_prefix_attention(*args, cache_pos=lens, workspace=torch.empty(256, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError, match="give one"):
        K.lora_delta(*_LORA, accumulate=True)
    with pytest.raises(nat.LeanB200Error):
        K.lora_delta(*_LORA, workspace=torch.empty(1, dtype=torch.uint8, device=DEV))
    # a parameter is a tensor like any other
    x = torch.nn.Parameter(_LORA[0], requires_grad=False)
    assert torch.equal(K.lora_delta(x, *_LORA[1:]), K.lora_delta(*_LORA))
