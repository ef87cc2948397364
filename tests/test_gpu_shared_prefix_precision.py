"""The probabilities of the attention behind a shared prefix, in every form, where their rounding would show.

One key in sixteen scores 0, the others -1: with the scale -ln p every other key
has the probability p = 0.5019, just below the middle of two bf16 (0.5 and 0.5 +
2^-8), and the values are such that the terms cancel.  The scores are
exact, so a probability is off by its own rounding (two bf16: 2^-16 of it) and by
the exponential's (2^-22, and 2^-24 of its argument): below 2^-15 in all; the fp32
sums of at most 2^10 terms of one sign each add less than 2^-14 of their
magnitude.  The output rounds to bf16 once.  So with A = sum p |v| / sum p

    |got - want| <= 2^-8 |want| + 2^-13 A.

One bf16 a probability gives 0.0033, fifteen times that tolerance.
"""

from __future__ import annotations

import math

import pytest
import torch

from leanstack_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


@pytest.mark.parametrize("batch,q_len,hq,hkv,prefix,own", [
    (2, 1, 16, 8, 300, 70),  # a few rows: the strips' kernel alone
    (32, 1, 32, 8, 1000, 40),  # decode: alternate key tiles
    (13, 5, 16, 8, 500, 60),  # verify
    (130, 1, 32, 8, 777, 20),  # 520 rows: shared key tiles
    (8, 100, 32, 8, 512, 130),  # prompts
    (1, 1, 8, 8, 0, 900),  # an own strip alone
])
def test_equal_probabilities_between_two_bf16(batch, q_len, hq, hkv, prefix, own):
    g, n = hq // hkv, own + q_len
    p = 0.5019
    scale = -math.log(p)
    gen = torch.Generator(device=DEV).manual_seed(3)
    q = torch.zeros(batch * q_len, hq, D, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 1.0

    def strip(*shape):  # [.., keys, D]
        k = torch.randn(*shape, D, generator=gen, device=DEV).bfloat16()
        top = torch.arange(shape[-1], device=DEV) % 16 == 0
        k[..., 0] = torch.where(top, 0.0, -1.0)
        v = torch.where(top, 15 * p, -1.0)[:, None] * (1 + torch.arange(D, device=DEV) % 3)
        return k, v.bfloat16().expand(*shape, D).contiguous()

    kp, vp = strip(hkv, max(prefix, 1))
    kc, vc = strip(batch, hkv, n)
    pos = torch.full((batch,), own, device=DEV, dtype=torch.int32)
    out = K.shared_prefix_attention(q, kp, vp, kc, vc, batch, q_len, hq, hkv, D, prefix, n, scale, cache_pos=pos)
    for i in range(q_len):  # every row of a step is the same but for the own keys that it sees
        k = torch.cat([kp[0, :prefix, 0], kc[0, 0, :own + i + 1, 0]]).double()
        v = torch.cat([vp[0, :prefix], vc[0, 0, :own + i + 1]]).double()
        w = torch.softmax(k * scale, 0)
        want, mag = w @ v, w @ v.abs()
        got = out.view(batch, q_len, hq, D)[:, i].double()
        worst = ((got - want).abs() - (want.abs() * 2 ** -8 + mag * 2 ** -13)).max().item()
        assert worst <= 0, f"token {i}: outside the tolerance by {worst:.3g}"
