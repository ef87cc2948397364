"""The groups of 8 logits that the token rules read lie inside the array, whatever the vocabulary (index arithmetic of
csrc/token_groups.cuh, compiled for the host)."""

from __future__ import annotations

import ctypes
import os
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "leanstack_b200" / "csrc"
SOURCE = """
#include "token_groups.cuh"
extern "C" {
int offset(long long row, long long V) { return lsb::tr_offset(row, V); }
int groups(int a, int V) { return lsb::tr_groups(a, V); }
int left(long long row, long long V, long long m) { return lsb::tr_left(row, V, m); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("groups")
    (d / "groups.cpp").write_text(SOURCE)
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC),
                    str(d / "groups.cpp"), "-o", str(d / "groups.so")], check=True)
    lib = ctypes.CDLL(str(d / "groups.so"))
    lib.offset.argtypes = [ctypes.c_longlong] * 2
    lib.left.argtypes = [ctypes.c_longlong] * 3
    return lib


@pytest.mark.parametrize("vocab", [*range(1, 34), 255, 1001])
def test_groups_cover_the_row_and_stay_inside(lib, vocab):
    for m in range(1, 18):
        for row in range(m):
            a, left = lib.offset(row, vocab), lib.left(row, vocab, m)
            base, n = row * vocab - a, lib.groups(a, vocab)
            assert base % 8 == 0
            assert 0 <= row * vocab - base < 8 and base + 8 * n >= (row + 1) * vocab
            for g in range(n):
                take = 8 if vocab % 8 == 0 or g * 8 + 8 <= left else left - g * 8  # what the kernel loads
                assert 0 < take <= 8 and base + 8 * g + take <= m * vocab, (m, row, g)
                assert g < n - 1 and take == 8 or base + 8 * g + take >= (row + 1) * vocab


def test_many_rows(lib):
    assert lib.left(0, (1 << 20) - 1, 65535) == 2 ** 31 - 1
    assert lib.left(65534, (1 << 20) - 1, 65535) == (1 << 20) - 1 + (65534 * ((1 << 20) - 1)) % 8


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", range(1, 8))
@pytest.mark.parametrize("m", [1, 3, 9])
def test_small_vocabularies(vocab, m):
    import torch

    from leanstack_b200 import kernels as K

    g = torch.Generator().manual_seed(vocab)
    for dtype in (torch.bfloat16, torch.float32):
        logits = torch.randn(m, vocab, generator=g).to("cuda", dtype)
        out = torch.empty(m, vocab, device="cuda")
        ids = K.constrained_argmax(logits, out_logits=out)
        assert torch.equal(out, logits.float()) and torch.equal(ids, logits.float().argmax(1))
