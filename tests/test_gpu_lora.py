"""Adapters of many requests at once against a 64-bit product.

Tolerance, per output element: whatever the order of the sums, an fp32 sum of
n products is off by at most n x 2^-24 of the sum of their magnitudes, so with
A = scaling sum_r |b| sum_k |a x| the two nested sums, the scaling and the
accumulation stay within (K + R + 4) x 2^-24 x A.
"""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(m, k, n, rank, adapters, seed=3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(m, k, generator=g, device=DEV).bfloat16()
    a = (torch.randn(adapters, rank, k, generator=g, device=DEV) * k ** -0.5).bfloat16()
    b = (torch.randn(adapters, n, rank, generator=g, device=DEV) * rank ** -0.5).bfloat16()
    s = torch.rand(adapters, generator=g, device=DEV) * 2 - 0.5
    return x, a, b, s


def _assert_close(got, x, a, b, s, ids, q_len, base=None):
    k, rank = x.shape[1], a.shape[1]
    want = torch.zeros(got.shape, dtype=torch.float64, device=DEV) if base is None else base.double()
    mag = want.abs()
    for i, ad in enumerate(ids):
        if 0 <= ad < a.shape[0]:
            rows = slice(i * q_len, (i + 1) * q_len)
            xd, ad_, bd = x[rows].double(), a[ad].double(), b[ad].double()
            want[rows] += float(s[ad]) * ((xd @ ad_.T) @ bd.T)
            mag[rows] += abs(float(s[ad])) * ((xd.abs() @ ad_.abs().T) @ bd.abs().T)
    err = (got.double() - want).abs()
    assert (err <= (k + rank + 4) * 2 ** -24 * mag).all(), (err / mag.clamp(min=1e-30)).max().item()
    none = [i for i, ad in enumerate(ids) if not 0 <= ad < a.shape[0]]
    for i in none:  # exactly nothing, and the base exactly itself
        rows = slice(i * q_len, (i + 1) * q_len)
        assert torch.equal(got[rows], torch.zeros_like(got[rows]) if base is None else base[rows])


@pytest.mark.parametrize("rank", [8, 16, 40, 64, 128])
@pytest.mark.parametrize("ids,q_len", [
    ([0], 1),
    ([-1], 1),
    ([2, 2, 2], 1),  # one adapter for all
    ([0, -1, 3, 1, 3, 2, 0, 4], 1),
    ([1, 0, -1, 1], 5),  # verify
    ([0, 4, 2], 40),  # prompts, ragged over any token tile
])
def test_matches_the_product(rank, ids, q_len):
    k, n, adapters = 264, 200, 5
    x, a, b, s = _inputs(len(ids) * q_len, k, n, rank, adapters)
    t = torch.tensor(ids, device=DEV, dtype=torch.int32)
    K.device_error(clear=True)
    out = torch.full((x.shape[0], n), float("nan"), device=DEV)
    assert K.lora_delta(x, a, b, s, t, q_len, out=out) is out
    _assert_close(out, x, a, b, s, ids, q_len)
    base = torch.randn_like(out)
    acc = base.clone()
    K.lora_delta(x, a, b, s, t, q_len, accumulate=True, out=acc)
    _assert_close(acc, x, a, b, s, ids, q_len, base)
    assert K.device_error(clear=True) == 0


@pytest.mark.parametrize("k,n", [(8, 8), (1024, 4096), (9728, 2560), (2560, 19456), (4096, 2568), (520, 136)])
@pytest.mark.parametrize("batch,q_len", [(1, 1), (33, 1), (128, 1), (7, 4), (2, 333)])
def test_projection_shapes(k, n, batch, q_len):
    adapters, rank = 6, 16
    ids = [(5 * i) % 7 - 1 for i in range(batch)]
    x, a, b, s = _inputs(batch * q_len, k, n, rank, adapters)
    out = K.lora_delta(x, a, b, s, torch.tensor(ids, device=DEV, dtype=torch.int32), q_len)
    _assert_close(out, x, a, b, s, ids, q_len)


def test_many_sequences_of_one_token_and_many_adapters():
    batch, k, n, rank, adapters = 700, 512, 264, 8, 300
    ids = [(i * 7) % 301 - 1 for i in range(batch)]
    x, a, b, s = _inputs(batch, k, n, rank, adapters)
    out = K.lora_delta(x, a, b, s, torch.tensor(ids, device=DEV, dtype=torch.int32))
    _assert_close(out, x, a, b, s, ids, 1)


def test_a_window_of_sequences_and_prompts_at_the_edges():
    """Sequences beyond the window that shares CTAs; the shortest prompts; token tiles that end inside."""
    for batch, q_len in ((1030, 1), (2100, 2), (3, 15), (3, 16), (2, 127), (2, 128), (1, 129), (5, 65)):
        ids = [(i * 3) % 5 - 1 for i in range(batch)]
        x, a, b, s = _inputs(batch * q_len, 256, 72, 24, 4)
        out = K.lora_delta(x, a, b, s, torch.tensor(ids, device=DEV, dtype=torch.int32), q_len)
        _assert_close(out, x, a, b, s, ids, q_len)


@pytest.mark.parametrize("batch", [1, 3, 15, 16, 40])
@pytest.mark.parametrize("n", [8, 120, 8192, 8200])
@pytest.mark.parametrize("rank", [8, 24, 64, 72])
def test_one_launch_and_two(batch, n, rank):
    """Few and many sequences, narrow and wide outputs, low and high ranks: every kernel and thread count."""
    k, adapters = 1064, 4
    ids = [(i * 3) % 5 - 1 if batch > 1 else 2 for i in range(batch)]
    x, a, b, s = _inputs(batch, k, n, rank, adapters)
    t = torch.tensor(ids, device=DEV, dtype=torch.int32)
    out = torch.full((batch, n), float("nan"), device=DEV)
    K.lora_delta(x, a, b, s, t, 1, out=out)
    _assert_close(out, x, a, b, s, ids, 1)
    base = torch.randn_like(out)
    acc = base.clone()
    K.lora_delta(x, a, b, s, t, 1, accumulate=True, out=acc)
    _assert_close(acc, x, a, b, s, ids, 1, base)


@pytest.mark.parametrize("rank", [16, 72])
@pytest.mark.parametrize("batch,q_len", [(80, 1), (35, 2), (30, 3), (14, 5), (11, 6), (9, 8), (7, 9), (5, 15)])
def test_tiles_of_one_adapter(batch, q_len, rank):
    """More tokens of one adapter than a tile holds, sequences that do not divide it, others in between."""
    k, n = 272, 136
    for ids in ([0] * batch, [0 if i % 3 else 1 - i % 2 * 2 for i in range(batch)]):
        x, a, b, s = _inputs(batch * q_len, k, n, rank, 2)
        x[0] = float("inf")  # stays with its token
        x[0, 1:] = 1.0
        out = K.lora_delta(x, a, b, s, torch.tensor(ids, device=DEV, dtype=torch.int32), q_len)
        x[0] = 0
        keep = out.clone()
        keep[0] = K.lora_delta(x, a, b, s, torch.tensor(ids, device=DEV, dtype=torch.int32), q_len)[0]
        _assert_close(keep, x, a, b, s, ids, q_len)
        assert ids[0] < 0 or not torch.isfinite(out[0]).any()


def test_an_unused_adapter_and_a_token_without_one_may_hold_anything():
    x, a, b, s = _inputs(3, 256, 256, 16, 4)
    a[1], b[1], s[1] = float("nan"), float("inf"), float("nan")
    x[1] = float("nan")
    ids = [0, -1, 3]
    out = K.lora_delta(x, a, b, s, torch.tensor(ids, device=DEV, dtype=torch.int32))
    assert torch.isfinite(out).all()
    x[1] = 0
    _assert_close(out, x, a, b, s, ids, 1)


def test_an_adapter_past_the_bank_is_reported_and_counts_as_none():
    x, a, b, s = _inputs(4, 256, 128, 8, 2)
    K.device_error(clear=True)
    ids = [0, 2, 1, 2 ** 31 - 1]
    out = K.lora_delta(x, a, b, s, torch.tensor(ids, device=DEV, dtype=torch.int32))
    assert K.device_error(clear=True) == 1  # LS_ERR_INVALID_ARGUMENT
    _assert_close(out, x, a, b, s, ids, 1)


@pytest.mark.parametrize("batch,q_len", [(9, 1), (2, 150)])
def test_same_bits_on_other_streams_workspaces_and_replays(batch, q_len):
    k, n, rank = 1024, 512, 16
    x, a, b, s = _inputs(batch * q_len, k, n, rank, 3)
    ids = torch.tensor([i % 4 - 1 for i in range(batch)], device=DEV, dtype=torch.int32)
    ws = torch.zeros(K.lora_delta_workspace_bytes(batch, q_len, k, n, rank), device=DEV, dtype=torch.uint8)
    want = K.lora_delta(x, a, b, s, ids, q_len, workspace=ws)
    for _ in range(3):
        assert torch.equal(K.lora_delta(x, a, b, s, ids, q_len, workspace=ws), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = K.lora_delta(x, a, b, s, ids, q_len)
    side.synchronize()
    assert torch.equal(again, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.lora_delta(x, a, b, s, ids, q_len, out=out, workspace=ws)
    for shift in (0, 1):  # other adapters without another capture
        ids2 = ids.roll(shift)
        want2 = K.lora_delta(x, a, b, s, ids2, q_len)
        ids.copy_(ids2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want2)


def test_adds_to_a_projection_as_one_more_partial():
    """gemm_tc_splits leaves its partials, lora_delta one more; the residual + RMSNorm consumer adds them all:
    bf16(residual + bf16(W x + delta)) within one rounding of each sum (2^-8) of the 64-bit result."""
    m, k, n, rank = 9, 1024, 512, 16
    x, a, b, s = _inputs(m, k, n, rank, 3)
    g = torch.Generator(device=DEV).manual_seed(8)
    w = (torch.randn(n, k, generator=g, device=DEV) * 0.03).bfloat16()
    res = torch.randn(m, n, generator=g, device=DEV).bfloat16()
    ids = [0, 1, 2, -1, 0, 1, 2, -1, 0]
    t = torch.tensor(ids, device=DEV, dtype=torch.int32)
    splits = K.gemm_splits(m, k, n)
    part = torch.zeros(splits + 1, m, n, device=DEV)
    assert K.gemm_tc_splits(x, w, part) == splits
    K.lora_delta(x, a, b, s, t, out=part[splits])
    out = torch.empty_like(res)
    K.residual_rmsnorm_splits(part, splits + 1, res, out_residual=out)
    y = x.double() @ w.double().T
    for i, ad in enumerate(ids):
        if ad >= 0:
            y[i] += float(s[ad]) * (b[ad].double() @ (a[ad].double() @ x[i].double()))
    want = res.double() + y
    tol = 2 ** -8 * (y.abs() + want.abs()) + 2 ** -15 * (1 + y.abs())
    assert ((out.double() - want).abs() <= tol).all()


def test_refusals():
    x, a, b, s = _inputs(4, 256, 128, 8, 2)
    ids = torch.zeros(4, device=DEV, dtype=torch.int32)
    K.lora_delta(x, a, b, s, ids)
    with pytest.raises(ValueError, match="not sequences of"):
        K.lora_delta(x, a, b, s, ids, 3)
    with pytest.raises(ValueError, match="adapter_ids must have shape"):
        K.lora_delta(x, a, b, s, ids, 2)
    with pytest.raises(ValueError, match="b must have shape"):
        K.lora_delta(x, a, b[:1], s, ids)
    with pytest.raises(TypeError, match="scaling"):
        K.lora_delta(x, a, b, s.bfloat16(), ids)
    with pytest.raises(TypeError, match="adapter_ids"):
        K.lora_delta(x, a, b, s, ids.long())
    with pytest.raises(ValueError, match="give one"):
        K.lora_delta(x, a, b, s, ids, accumulate=True)
    with pytest.raises(TypeError, match="out"):
        K.lora_delta(x, a, b, s, ids, out=torch.empty(4, 128, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(K.nat.LeanB200Error, match="multiples of 8"):
        K.lora_delta(x, a[:, :4].contiguous(), b[..., :4].contiguous(), s, ids)
    with pytest.raises(K.nat.LeanB200Error, match="workspace needs"):
        K.lora_delta(x, a, b, s, ids, workspace=torch.zeros(16, device=DEV, dtype=torch.uint8))
