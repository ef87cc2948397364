"""The C++ front end of the multi-request calls leaves every operand that is not plainly right to the Python checks
(no GPU needed: it answers None before anything is enqueued)."""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import _native as nat
from leanstack_b200 import kernels as K

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def front():
    if not nat.LIB_PATH.exists() or not nat.FRONT_PATH.exists():
        from leanstack_b200 import build

        build.build()
    return nat.front()


def _prefix_args():
    kv = torch.zeros(2, 64, 128, dtype=BF16)
    cache = torch.zeros(3, 2, 16, 128, dtype=BF16)
    q = torch.zeros(3, 8 * 128, dtype=BF16)
    return [q, kv, kv, cache, cache, 3, 1, 8, 2, 128, 50, 16, 0.088, torch.zeros(3, dtype=torch.int32), 0, None, None]


def _lora_args():
    return [torch.zeros(4, 64, dtype=BF16), torch.zeros(2, 8, 64, dtype=BF16), torch.zeros(2, 32, 8, dtype=BF16),
            torch.ones(2), torch.zeros(4, dtype=torch.int32), 1, False, None, None]


def _rules_args():
    return [torch.zeros(2, 64), *[None] * 8, False, None, None, None]


@pytest.mark.parametrize("name,make", [("shared_prefix_attention", _prefix_args), ("lora_delta", _lora_args),
                                       ("constrained_argmax", _rules_args)])
def test_not_plainly_right_is_not_taken(front, name, make):
    fn = getattr(front, name)
    good = make()
    assert fn(*good) is None  # tensors of the host
    assert fn() is None and fn(*good[:-1]) is None and fn(*good, None) is None
    for i in range(len(good)):
        for bad in (None, "x", -1, 1 << 40, 1 << 80, 1.5, [1], True, torch.zeros(()), torch.zeros(0, 5)):
            args = list(good)
            args[i] = bad
            assert fn(*args) is None, (i, bad)


def test_the_python_checks_name_the_fault(front):
    with pytest.raises(ValueError, match="CUDA tensor"):
        K.shared_prefix_attention(*_prefix_args()[:13], cache_pos=_prefix_args()[13])
    with pytest.raises(ValueError, match="CUDA tensor"):
        K.lora_delta(*_lora_args()[:5])
    with pytest.raises(ValueError, match="CUDA tensor"):
        K.constrained_argmax(_rules_args()[0])
    with pytest.raises(TypeError, match="bf16 or fp32"):
        K.constrained_argmax(torch.zeros(2, 64, dtype=torch.int32))


def test_a_status_becomes_an_error(front):
    with pytest.raises(nat.LeanB200Error, match="LS_ERR_KV_OVERFLOW"):
        nat.finished("ls_shared_prefix_attention", 6)
    out = torch.zeros(1)
    assert nat.finished("ls_lora_delta", out) is out


def test_missing_front_fails_loudly(front, monkeypatch, tmp_path):
    monkeypatch.setattr(nat, "FRONT_PATH", tmp_path / "nope.so")
    monkeypatch.setattr(nat, "_FRONT", None)
    with pytest.raises(nat.NativeLibraryMissing):
        K.lora_delta(*_lora_args()[:5])
