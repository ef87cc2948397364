"""Attention behind a shared prefix against a 64-bit softmax over prefix and cache.

Tolerance, per output element: the output rounds to bf16 once (2^-8 of its
value); the probabilities may enter the value product as bf16 (2^-8 of each
term, so at most 2^-8 of A = sum p |v| / sum p); scores are fp32 dot products
of 128 terms (error below 128 x 2^-24 x sum |q k| x scale, under 2^-13 for the
unit-variance inputs here, where sum |q k| x scale stays below 16), so each
probability is off by less than 2^-12 of itself.
"""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


def _inputs(batch, q_len, hq, hkv, prefix, cap, slots, seed=5):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def n(*shape):
        return torch.randn(shape, generator=g, device=DEV).bfloat16()

    return n(batch * q_len, hq, D), n(hkv, cap, D), n(hkv, cap, D), n(batch, hkv, slots, D), n(batch, hkv, slots, D)


def _reference(q, kp, vp, kc, vc, lens, batch, q_len, hq, hkv, prefix, scale):
    """(attention, sum p |v| / sum p) in float64, one sequence and kv head at a time."""
    g = hq // hkv
    qs = q.view(batch, q_len, hq, D).double()
    out = torch.empty(batch, q_len, hq, D, dtype=torch.float64, device=q.device)
    mag = torch.empty_like(out)
    for b in range(batch):
        n = lens[b] + q_len
        later = torch.arange(n, device=q.device)[None] > (lens[b] + torch.arange(q_len, device=q.device))[:, None]
        later = torch.cat([torch.zeros(q_len, prefix, dtype=torch.bool, device=q.device), later], 1)
        for h in range(hkv):
            k = torch.cat([kp[h, :prefix], kc[b, h, :n]]).double()
            v = torch.cat([vp[h, :prefix], vc[b, h, :n]]).double()
            s = torch.einsum("qgd,kd->gqk", qs[b, :, h * g:(h + 1) * g], k) * scale
            w = torch.softmax(s.masked_fill(later, float("-inf")), -1)
            out[b, :, h * g:(h + 1) * g] = (w @ v).transpose(0, 1)
            mag[b, :, h * g:(h + 1) * g] = (w @ v.abs()).transpose(0, 1)
    return out.view(batch * q_len, -1), mag.view(batch * q_len, -1)


def _assert_close(got, want, mag):
    got = got.double()
    assert torch.isfinite(got).all()
    tol = want.abs() * 2 ** -8 + mag * (2 ** -8 + 2 ** -12)
    worst = ((got - want).abs() - tol).max().item()
    assert worst <= 0, f"outside the tolerance by {worst:.3g}"


def _check(batch, q_len, hq, hkv, prefix, lens, slots, cap=None, poison=True):
    cap = prefix if cap is None else cap
    q, kp, vp, kc, vc = _inputs(batch, q_len, hq, hkv, prefix, cap, slots)
    if poison:  # memory behind the prefix and behind every sequence is the caller's
        kp[:, prefix:] = float("nan")
        vp[:, prefix:] = float("nan")
        for b in range(batch):
            kc[b, :, lens[b] + q_len:] = float("nan")
            vc[b, :, lens[b] + q_len:] = float("inf")
    pos = torch.tensor(lens, device=DEV, dtype=torch.int32)
    scale = D ** -0.5
    K.device_error(clear=True)
    out = K.shared_prefix_attention(q, kp, vp, kc, vc, batch, q_len, hq, hkv, D, prefix, slots, scale, cache_pos=pos)
    want, mag = _reference(q, kp, vp, kc, vc, lens, batch, q_len, hq, hkv, prefix, scale)
    assert K.device_error(clear=True) == 0
    _assert_close(out, want, mag)
    return out


@pytest.mark.parametrize("hq,hkv", [(32, 8), (16, 8), (8, 2), (5, 5), (24, 1)])
@pytest.mark.parametrize("batch,q_len,prefix,lens,slots", [
    (1, 1, 1, [0], 1),  # one key each
    (2, 1, 0, [0, 9], 16),  # no prefix
    (3, 1, 63, [0, 15, 16], 32),  # ends inside a key tile
    (3, 1, 64, [1, 2, 40], 41),  # ends on one; the last slot in use
    (2, 5, 130, [0, 77], 96),  # verify
    (5, 3, 1000, [511, 0, 100, 3, 4], 515),
])
def test_decode_and_verify_rows(hq, hkv, batch, q_len, prefix, lens, slots):
    _check(batch, q_len, hq, hkv, prefix, lens, slots)


@pytest.mark.parametrize("batch,q_len,hq,hkv,prefix,slots", [
    (32, 1, 32, 8, 4100, 300),  # 128 rows per kv head: one full row tile
    (33, 1, 32, 8, 777, 70),  # one row tile and 4 rows
    (16, 5, 32, 8, 2049, 200),  # 320 rows
    (100, 1, 8, 8, 515, 40),  # 100 rows
    (2, 70, 32, 8, 500, 128),  # 280 rows per sequence and kv head: prompts
    (3, 129, 16, 8, 333, 200),
    (1, 300, 8, 2, 0, 301),  # a prompt without a prefix
    (8, 100, 32, 8, 700, 260),  # prompts that fill the GPU by their rows: 400 rows per sequence and kv head
    (20, 140, 16, 8, 129, 200),
    (9, 65, 32, 8, 0, 130),
    (40, 257, 8, 4, 64, 300),
])
def test_wide_batches_and_prompts(batch, q_len, hq, hkv, prefix, slots):
    lens = [(37 * b) % max(1, slots - q_len) for b in range(batch)]
    _check(batch, q_len, hq, hkv, prefix, lens, slots, cap=prefix + 13)


@pytest.mark.parametrize("batch,q_len,hq,hkv", [(1, 1, 8, 8), (4, 1, 32, 8), (1, 4, 8, 2), (2, 2, 8, 2), (16, 1, 2, 2),
                                                (5, 1, 6, 2), (17, 1, 2, 2)])
@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 2047, 2048, 2049])
def test_few_rows(batch, q_len, hq, hkv, prefix):
    """Around the sizes at which the prefix goes to the strips' kernel; own strips shorter and longer than it."""
    _check(batch, q_len, hq, hkv, prefix, [(37 * i) % (300 - q_len) for i in range(batch)], 300)
    _check(batch, q_len, hq, hkv, prefix, [0] * batch, q_len)


@pytest.mark.parametrize("batch,q_len,hq,hkv,prefix", [(1, 251, 32, 8, 6985), (3, 80, 32, 8, 3001), (130, 1, 32, 8, 5000),
                                                       (20, 8, 16, 2, 2500)])
def test_row_mode_gives_the_same_bits_every_time(batch, q_len, hq, hkv, prefix):
    """Two streams share the K/V ring and stage their partials in it: neither before the other is done."""
    lens = [(5 * i) % 17 for i in range(batch)]
    first = _check(batch, q_len, hq, hkv, prefix, lens, 17 + q_len)
    for _ in range(20):
        assert torch.equal(_check(batch, q_len, hq, hkv, prefix, lens, 17 + q_len), first)


def test_workspace_grows_with_the_prefix():
    for batch, q_len, hq, hkv in ((1, 1, 8, 8), (4, 1, 32, 8), (16, 1, 2, 2), (17, 1, 2, 2), (3, 5, 32, 8)):
        need = [K.shared_prefix_attention_workspace_bytes(batch, q_len, hq, hkv, 128, p)
                for p in (0, 1, 100, 500, 1000, 2047, 2048, 2049, 2100, 3000, 9000, 30000)]
        assert need == sorted(need), (batch, q_len, need)


def test_long_prefix():
    _check(4, 1, 16, 8, 70001, [3, 0, 50, 17], 64, cap=70003)


def test_peaked_scores_and_rescaling():
    """Scores that grow along the prefix by far more than the softmax's range: the running maximum moves in every tile."""
    batch, hq, hkv, prefix, slots = 2, 8, 2, 900, 32
    q, kp, vp, kc, vc = _inputs(batch, 1, hq, hkv, prefix, prefix, slots)
    q[:] = 1.0
    kp[:] = (torch.arange(prefix, device=DEV) / prefix).bfloat16()[None, :, None]
    kc[:] = -3.0
    scale = D ** -0.5
    pos = torch.tensor([5, 31], device=DEV, dtype=torch.int32)
    out = K.shared_prefix_attention(q, kp, vp, kc, vc, batch, 1, hq, hkv, D, prefix, slots, scale, cache_pos=pos)
    want, mag = _reference(q, kp, vp, kc, vc, [5, 31], batch, 1, hq, hkv, prefix, scale)
    _assert_close(out, want, mag)


def test_minus_infinity_keys_are_left_out():
    """Keys whose score is -inf for every row (a poisoned half of the prefix) get no weight; the rest stays right."""
    batch, hq, hkv, prefix, slots = 3, 8, 2, 200, 16
    q, kp, vp, kc, vc = _inputs(batch, 1, hq, hkv, prefix, prefix, slots)
    q[..., 0] = 1.0
    kp[:, :128] = 0.0
    kp[:, :128, 0] = float("-inf")
    scale = D ** -0.5
    pos = torch.tensor([1, 2, 3], device=DEV, dtype=torch.int32)
    out = K.shared_prefix_attention(q, kp, vp, kc, vc, batch, 1, hq, hkv, D, prefix, slots, scale, cache_pos=pos)
    want, mag = _reference(q, kp, vp, kc, vc, [1, 2, 3], batch, 1, hq, hkv, prefix, scale)
    _assert_close(out, want, mag)


@pytest.mark.parametrize("batch,q_len,prefix", [(4, 1, 600), (1, 200, 300)])
def test_uniform_cursor_streams_and_replay(batch, q_len, prefix):
    """The host cursor, a side stream and a captured graph replayed on changed inputs give the same bits."""
    hq, hkv, slots = 16, 8, 256
    q, kp, vp, kc, vc = _inputs(batch, q_len, hq, hkv, prefix, prefix, slots)
    scale = D ** -0.5
    args = (batch, q_len, hq, hkv, D, prefix, slots, scale)
    pos = torch.full((batch,), 20, device=DEV, dtype=torch.int32)
    ws = torch.zeros(max(256, K.shared_prefix_attention_workspace_bytes(batch, q_len, hq, hkv, D, prefix)), device=DEV,
                     dtype=torch.uint8)
    want = K.shared_prefix_attention(q, kp, vp, kc, vc, *args, cache_pos=pos, workspace=ws)
    assert torch.equal(K.shared_prefix_attention(q, kp, vp, kc, vc, *args, uniform_past=20, workspace=ws), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = K.shared_prefix_attention(q, kp, vp, kc, vc, *args, cache_pos=pos)
    side.synchronize()
    assert torch.equal(again, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.shared_prefix_attention(q, kp, vp, kc, vc, *args, cache_pos=pos, out=out, workspace=ws)
    for shift in (0, 7):
        q2 = q.roll(shift, 0) * (1 + shift)
        pos2 = pos - shift
        want2 = K.shared_prefix_attention(q2, kp, vp, kc, vc, *args, cache_pos=pos2)
        q.copy_(q2)
        pos.copy_(pos2)
        for _ in range(2):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want2)


@pytest.mark.parametrize("q_len", [1, 90])
def test_cursor_outside_the_cache_is_reported(q_len):
    """A sequence whose cursor leaves its cache raises the device flag and reads nothing outside; the others are untouched."""
    hq, hkv, prefix, slots, batch = 8, 2, 100, 96, 3
    q, kp, vp, kc, vc = _inputs(batch, q_len, hq, hkv, prefix, prefix, slots)
    scale = D ** -0.5
    good = torch.tensor([3, 3, 3], device=DEV, dtype=torch.int32)
    want = K.shared_prefix_attention(q, kp, vp, kc, vc, batch, q_len, hq, hkv, D, prefix, slots, scale, cache_pos=good)
    K.device_error(clear=True)
    for bad in (slots, 2 ** 31 - 1, -1, -2 ** 31):
        pos = torch.tensor([3, bad, 3], device=DEV, dtype=torch.int32)
        out = K.shared_prefix_attention(q, kp, vp, kc, vc, batch, q_len, hq, hkv, D, prefix, slots, scale,
                                        cache_pos=pos)
        assert K.device_error(clear=True) == 6  # LS_ERR_KV_OVERFLOW
        assert torch.isfinite(out).all()
        assert torch.equal(out[:q_len], want[:q_len]) and torch.equal(out[2 * q_len:], want[2 * q_len:])
    # no prefix and no key of its own: zeros
    pos = torch.tensor([3, -q_len, 3], device=DEV, dtype=torch.int32)
    out = K.shared_prefix_attention(q, kp, vp, kc, vc, batch, q_len, hq, hkv, D, 0, slots, scale, cache_pos=pos)
    assert K.device_error(clear=True) == 6
    assert not out[q_len:2 * q_len].any()


def test_refusals():
    hq, hkv, prefix, slots, batch = 8, 2, 100, 32, 2
    q, kp, vp, kc, vc = _inputs(batch, 1, hq, hkv, prefix, prefix, slots)
    pos = torch.zeros(batch, device=DEV, dtype=torch.int32)

    def call(q=q, kp=kp, vp=vp, kc=kc, vc=vc, prefix=prefix, slots=slots, **kw):
        kw.setdefault("cache_pos", pos)
        return K.shared_prefix_attention(q, kp, vp, kc, vc, batch, 1, hq, hkv, D, prefix, slots, D ** -0.5, **kw)

    call()
    with pytest.raises(K.nat.LeanB200Error, match="beyond prefix_cap"):
        call(prefix=prefix + 1)
    with pytest.raises(K.nat.LeanB200Error, match="beyond max_seq"):
        call(cache_pos=None, uniform_past=slots)
    with pytest.raises(TypeError, match="k_prefix"):
        call(kp=kp.half())
    with pytest.raises(ValueError, match="v_prefix must have shape"):
        call(vp=vp[:, :50].contiguous())
    with pytest.raises(ValueError, match="contiguous"):
        call(kc=kc.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(ValueError, match="k_cache must have shape"):
        call(slots=slots - 1)
    with pytest.raises(ValueError, match="q holds"):
        call(q=q[:1])
    with pytest.raises(ValueError, match="cache_pos must have shape"):
        call(cache_pos=pos[:1])
    with pytest.raises(TypeError, match="cache_pos"):
        call(cache_pos=pos.long())
    with pytest.raises(ValueError, match="CUDA tensor"):
        call(kc=kc.cpu())
