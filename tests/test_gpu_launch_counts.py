"""kernel_launches_per_step against the kernel nodes of a captured decode step."""

from __future__ import annotations

import ctypes

import pytest
import torch

from leanstack_b200 import kernels as K
from leanstack_b200 import synth
from leanstack_b200.config import TINY
from leanstack_b200.engine import DecodeEngine
from leanstack_b200.leanserve import materialize_from_tensors
from leanstack_b200.requests import AdapterBank, TokenRules

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def runtime():
    return materialize_from_tensors(TINY, {k: v.to(DEV) for k, v in synth.synth_checkpoint(TINY, 3).items()}, device=DEV)


def _kernel_nodes(eng) -> int:
    eng._decode_once()  # attributes set, symbols resolved
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        eng._decode_once()
    rt = ctypes.CDLL("libcudart.so.12")
    raw, n = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert rt.cudaGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert rt.cudaGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    kernels = 0
    for node in nodes:
        kind = ctypes.c_int(-1)
        assert rt.cudaGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        kernels += kind.value == 0  # cudaGraphNodeTypeKernel
    return kernels


@pytest.mark.parametrize("rules", [False, True])
@pytest.mark.parametrize("rank", [0, 16, 128])
@pytest.mark.parametrize("prefix", [0, 40, 300])
@pytest.mark.parametrize("batch,backend", [(1, "cuda_core"), (1, "tc"), (3, "cuda_core"), (4, "tc"), (20, "tc"), (40, "tc")])
def test_decode_step(runtime, batch, backend, prefix, rank, rules):
    if rank and backend == "cuda_core":
        pytest.skip("adapters run beside the tc linears")
    bank = AdapterBank(TINY, 2, rank, DEV) if rank else None
    eng = DecodeEngine(runtime, batch, 64, linear_backend=backend, prefix_capacity=prefix, adapters=bank,
                       rules=TokenRules(batch, TINY.vocab_size, DEV) if rules else None)
    if prefix:
        eng.prefill_prefix(synth.token_ids((prefix,), TINY.vocab_size, 3, "count/prefix"))
    eng.prefill(synth.token_ids((batch, 5), TINY.vocab_size, 3, "count/prompt").to(DEV))
    assert _kernel_nodes(eng) == eng.kernel_launches_per_step()


def _launches(call) -> int:
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    rt = ctypes.CDLL("libcudart.so.12")
    n = ctypes.c_size_t(0)
    assert rt.cudaGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("batch,q_len,hq,hkv", [(1, 1, 8, 8), (4, 1, 32, 8), (5, 1, 32, 8), (13, 5, 16, 8), (130, 1, 32, 8),
                                                (8, 100, 32, 8), (2, 70, 32, 8)])
@pytest.mark.parametrize("prefix", [0, 1, 2048, 2049])
def test_attention_calls(batch, q_len, hq, hkv, prefix):
    def z(*shape):
        return torch.zeros(shape, device=DEV, dtype=torch.bfloat16)

    q, kp, kc = z(batch * q_len, hq, 128), z(hkv, max(prefix, 1), 128), z(batch, hkv, q_len + 9, 128)
    ws = torch.zeros(max(256, K.shared_prefix_attention_workspace_bytes(batch, q_len, hq, hkv, 128, prefix)), device=DEV,
                     dtype=torch.uint8)
    out = z(batch * q_len, hq * 128)
    assert K.shared_prefix_attention_launches(batch, q_len, hq, hkv, 128, prefix) == _launches(
        lambda: K.shared_prefix_attention(q, kp, kp, kc, kc, batch, q_len, hq, hkv, 128, prefix, q_len + 9, 0.1,
                                          uniform_past=9, out=out, workspace=ws))


@pytest.mark.parametrize("batch,q_len", [(1, 1), (31, 1), (32, 1), (2, 15), (2, 16)])
@pytest.mark.parametrize("n", [64, 8192, 8200])
@pytest.mark.parametrize("rank", [8, 32, 40, 64, 72])
def test_adapter_calls(batch, q_len, n, rank):
    x = torch.zeros(batch * q_len, 256, device=DEV, dtype=torch.bfloat16)
    a, b = (torch.zeros(1, *s, device=DEV, dtype=torch.bfloat16) for s in ((rank, 256), (n, rank)))
    scaling, ids = torch.ones(1, device=DEV), torch.zeros(batch, device=DEV, dtype=torch.int32)
    out = torch.empty(batch * q_len, n, device=DEV)
    ws = torch.empty(K.lora_delta_workspace_bytes(batch, q_len, 256, n, rank), device=DEV, dtype=torch.uint8)
    assert K.lora_delta_launches(batch, q_len, 256, n, rank) == _launches(
        lambda: K.lora_delta(x, a, b, scaling, ids, q_len, out=out, workspace=ws))
