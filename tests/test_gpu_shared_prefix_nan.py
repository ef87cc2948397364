"""NaN and infinities that a row of the shared-prefix attention sees come out as NaN, in every form; other rows keep
their values.  Which outputs are NaN follows from the formula in 64 bits; the finite ones stay within the tolerance
of test_gpu_shared_prefix.py."""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import kernels as K
from test_gpu_shared_prefix import D, DEV, _inputs, _reference

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("batch,q_len,hq,hkv,prefix,own", [
    (2, 1, 16, 8, 300, 70),  # a few rows: the strips' kernel alone
    (32, 1, 32, 8, 1000, 40),  # decode: alternate key tiles
    (13, 5, 16, 8, 500, 60),  # verify
    (130, 1, 32, 8, 777, 20),  # 520 rows: shared key tiles
    (8, 100, 32, 8, 512, 130),  # prompts
    (3, 1, 8, 8, 0, 200),  # own strips alone
])
@pytest.mark.parametrize("where", ["k_prefix nan", "k_prefix inf", "k_own nan", "k_own inf", "query", "v_prefix", "v_own",
                                   "v light"])
def test_what_is_not_finite_shows(where, batch, q_len, hq, hkv, prefix, own):
    if prefix == 0 and where.startswith(("k_prefix", "v_prefix")):
        pytest.skip("no prefix")
    q, kp, vp, kc, vc = _inputs(batch, q_len, hq, hkv, prefix, max(prefix, 1), own + q_len)
    last = batch - 1
    if where == "k_prefix nan":
        kp[1, prefix // 2, 5] = NAN
    elif where == "k_prefix inf":  # a score of +inf or -inf, as the query's sign has it
        kp[1, prefix // 2, 5] = INF
    elif where == "k_own nan":
        kc[last, 0, own // 2, 7] = NAN
    elif where == "k_own inf":
        kc[last, 0, own // 2, 7] = INF
    elif where == "query":  # every score of the row
        q[-1, 1, 0] = NAN
    elif where == "v_prefix":
        vp[0, prefix - 1, 9] = NAN
    elif where == "v_own":
        vc[last, 0, 0, 100] = INF
    else:  # a value whose weight is below the smallest float: 0 x NaN is NaN
        q[..., 0] = 4.0
        kc[:, :, 0, 0] = -4000.0
        vc[last, 0, 0, 3] = NAN
    scale = D ** -0.5
    pos = torch.full((batch,), own, device=DEV, dtype=torch.int32)
    out = K.shared_prefix_attention(q, kp, vp, kc, vc, batch, q_len, hq, hkv, D, prefix, own + q_len, scale, cache_pos=pos)
    want, mag = _reference(q, kp, vp, kc, vc, [own] * batch, batch, q_len, hq, hkv, prefix, scale)
    bad = ~torch.isfinite(want)
    assert not bad.all() and (bad.any() or where.endswith("inf"))  # (-inf in every row that sees it: no weight, no NaN)
    got = out.double()
    assert torch.equal(~torch.isfinite(got), bad)
    err = (got - want).masked_fill(bad, 0.0).abs()
    tol = (want.abs() * 2 ** -8 + mag * (2 ** -8 + 2 ** -12)).masked_fill(bad, 0.0)
    assert (err <= tol).all()
