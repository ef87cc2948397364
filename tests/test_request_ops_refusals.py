"""The multi-request operators refuse bad arguments with a status code before any CUDA call (no GPU needed:
the addresses below are never dereferenced)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from leanstack_b200 import _native as nat
from leanstack_b200 import kernels as K

P = 256  # a 16-byte aligned stand-in address
F = ctypes.c_float(0.088)


@pytest.fixture(scope="module")
def lib():
    if not nat.LIB_PATH.exists():
        from leanstack_b200 import build

        build.build()
    return nat.load()


def _refused(fn, args, changes, code):
    a = list(args)
    for i, v in changes.items():
        a[i] = v
    assert fn(*a) == code, (changes, nat.last_error())


def test_shared_prefix_attention(lib):
    #        q  kp vp len  cap  kc vc pos past batch q_len hq hkv D max_seq scale out ws bytes stream
    args = [P, P, P, 500, 512, P, P, P, 0, 4, 1, 32, 8, 128, 64, F, P, P, 1 << 40, None]
    fn = lib.ls_shared_prefix_attention
    for changes, code in (({0: None}, 1), ({16: None}, 1), ({1: None}, 1), ({9: 0}, 1), ({10: 0}, 1), ({11: 30}, 1),
                          ({12: 0}, 1), ({14: 0}, 1), ({3: -1}, 1), ({13: 64}, 2), ({0: P + 2}, 3), ({2: P + 8}, 3),
                          ({3: 513}, 6), ({7: None, 8: 64}, 6), ({7: None, 8: -1}, 6)):
        _refused(fn, args, changes, code)
    n = ctypes.c_int64(0)
    assert lib.ls_shared_prefix_attention_workspace_bytes(4, 1, 32, 8, 128, 500, None) == 1
    assert lib.ls_shared_prefix_attention_workspace_bytes(4, 1, 32, 8, 64, 500, ctypes.byref(n)) == 2


def test_lora_delta(lib):
    #       x batch q_len k   a  b scaling adapters n rank ids acc out ws bytes stream
    args = [P, 4, 1, 2560, P, P, P, 8, 6144, 16, P, 0, P, P, 1 << 40, None]
    fn = lib.ls_lora_delta
    for changes, code in (({0: None}, 1), ({4: None}, 1), ({10: None}, 1), ({12: None}, 1), ({1: 0}, 1), ({2: 0}, 1),
                          ({7: 0}, 1), ({9: 0}, 1), ({9: 136}, 2), ({3: 2564}, 3), ({8: 6146}, 3), ({9: 12}, 3),
                          ({0: P + 4}, 3), ({13: None}, 4), ({14: 16}, 4)):
        _refused(fn, args, changes, code)


def test_constrained_argmax(lib):
    #       logits f32 m vocab counts seen rep freq pres bias_ids bias_vals cap allowed record out logits ws bytes stream
    args = [P, 0, 4, 151936, P, P, P, P, P, P, P, 3, P, 1, P, P, P, 1 << 40, None]
    fn = lib.ls_constrained_argmax
    for changes, code in (({0: None}, 1), ({14: None}, 1), ({2: 0}, 1), ({3: 0}, 1), ({4: None}, 1), ({5: None}, 1),
                          ({4: None, 5: None}, 1), ({9: None}, 1), ({11: 0}, 1), ({3: (1 << 21) + 1}, 2),
                          ({0: P + 2}, 3), ({15: P + 4}, 3), ({16: None}, 4), ({17: 8}, 4)):
        _refused(fn, args, changes, code)
    fn = lib.ls_token_stats_add
    args = [P, 4, 10, 1000, P, P, None]
    for changes, code in (({0: None}, 1), ({5: None}, 1), ({1: 0}, 1), ({2: 0}, 1), ({3: 0}, 1), ({3: (1 << 21) + 1}, 1)):
        _refused(fn, args, changes, code)


def test_constrained_argmax_bounds_its_bias_lists(lib):
    """Every bias meets every other of its row: a list that would keep the GPU for long is refused."""
    args = [P, 0, 4, 151936, None, None, None, None, None, P, P, (1 << 14) + 1, None, 0, P, None, P, 1 << 40, None]
    assert lib.ls_constrained_argmax(*args) == 2, nat.last_error()


def test_front_end_refuses_cpu_tensors():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    kv = torch.zeros(2, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU path"):
        K.shared_prefix_attention(x.view(2, 2, 128), kv, kv, kv[None], kv[None], 1, 2, 2, 2, 128, 16, 16, 0.1)
    with pytest.raises(ValueError, match="no CPU path"):
        K.lora_delta(x, torch.zeros(1, 8, 256, dtype=torch.bfloat16), torch.zeros(1, 8, 8, dtype=torch.bfloat16),
                     torch.ones(1), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="no CPU path"):
        K.constrained_argmax(x)
    with pytest.raises(ValueError, match="no CPU path"):
        K.token_stats_add(torch.zeros(1, 4, dtype=torch.int64), torch.zeros(1, 4, dtype=torch.int32), 100)
