"""A negative or zero scale of the shared-prefix attention, in every form: the tolerance of test_gpu_shared_prefix.py."""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import kernels as K
from test_gpu_shared_prefix import D, DEV, _assert_close, _inputs, _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [-D ** -0.5, 0.0, -1.0, 1e-3])
@pytest.mark.parametrize("batch,q_len,hq,hkv,prefix,own", [
    (2, 1, 16, 8, 300, 70),  # a few rows: the strips' kernel alone
    (32, 1, 32, 8, 1000, 40),  # decode: alternate key tiles
    (13, 5, 16, 8, 500, 60),  # verify
    (130, 1, 32, 8, 777, 20),  # 520 rows: shared key tiles
    (8, 100, 32, 8, 512, 130),  # prompts
    (3, 1, 8, 8, 0, 200),  # own strips alone
])
def test_any_sign(scale, batch, q_len, hq, hkv, prefix, own):
    q, kp, vp, kc, vc = _inputs(batch, q_len, hq, hkv, prefix, max(prefix, 1), own + q_len)
    if scale == -1.0:  # scores as far apart as the usual scale's: 1 / sqrt(D) of them in the query
        q = (q.float() * D ** -0.5).bfloat16()
    pos = torch.full((batch,), own, device=DEV, dtype=torch.int32)
    out = K.shared_prefix_attention(q, kp, vp, kc, vc, batch, q_len, hq, hkv, D, prefix, own + q_len, scale, cache_pos=pos)
    want, mag = _reference(q, kp, vp, kc, vc, [own] * batch, batch, q_len, hq, hkv, prefix, scale)
    _assert_close(out, want, mag)
