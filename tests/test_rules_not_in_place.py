"""constrained_argmax refuses processed logits that overlap the logits it reads."""

from __future__ import annotations

import pytest
import torch

from leanstack_b200 import _native as nat
from leanstack_b200 import kernels as K

P = 1 << 20
M, VOCAB = 4, 1000


@pytest.fixture(scope="module")
def lib():
    if not nat.LIB_PATH.exists():
        from leanstack_b200 import build

        build.build()
    return nat.load()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are no memory: for a machine without a GPU")
@pytest.mark.parametrize("f32", [0, 1])
def test_overlap_is_refused(lib, f32):
    size = M * VOCAB * (4 if f32 else 2)
    for at in (P, P + 16, P + size - 16, P - 16, P - M * VOCAB * 4 + 16):
        rc = lib.ls_constrained_argmax(P, f32, M, VOCAB, None, None, None, None, None, None, None, 0, None, 0, 256, at,
                                       256, 1 << 20, None)
        assert rc == 1, (at - P, nat.last_error())  # LS_ERR_INVALID_ARGUMENT
        assert "overlaps" in nat.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_in_place_is_refused_and_next_to_it_is_not(dtype):
    size = dtype.itemsize
    room = torch.empty(M * VOCAB * (4 + size + 4), dtype=torch.uint8, device="cuda")
    before, logits, behind = room.split([M * VOCAB * 4, M * VOCAB * size, M * VOCAB * 4])
    logits = logits.view(dtype).view(M, VOCAB)
    logits.copy_(torch.randn(M, VOCAB, generator=torch.Generator().manual_seed(1)))
    kept = logits.clone()
    over = room[M * VOCAB * 4 - 64:M * VOCAB * 8 - 64].view(torch.float32).view(M, VOCAB)
    for out in [over] + ([logits] if dtype is torch.float32 else []):
        with pytest.raises(nat.LeanB200Error, match="overlaps"):
            K.constrained_argmax(logits, out_logits=out)
    for out in (before, behind):
        out = out.view(torch.float32).view(M, VOCAB)
        ids = K.constrained_argmax(logits, out_logits=out)
        assert torch.equal(out, kept.float()) and torch.equal(ids, kept.float().argmax(1))
    assert torch.equal(logits, kept)
