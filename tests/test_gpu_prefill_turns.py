"""Calls of the gated delta rule over sequences that are worked off in turns: how they are cut."""

import ctypes

import pytest
import torch

from carrykernel_b200.vllm_integration import packed_prefill as pp
from test_gpu_prefill import BF16, DEV, make, run, starts

pytestmark = pytest.mark.gpu


class KernelNode(ctypes.Structure):
    _fields_ = [("func", ctypes.c_void_p), ("grid", ctypes.c_uint * 3), ("block", ctypes.c_uint * 3), ("shared", ctypes.c_uint),
                ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p), ("kernel", ctypes.c_void_p), ("context", ctypes.c_void_p)]


def ctas_of(graph):
    """CTAs of all kernels of a captured graph."""
    driver, raw, count = ctypes.CDLL("libcuda.so.1"), ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    assert driver.cuGraphGetNodes(raw, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert driver.cuGraphGetNodes(raw, nodes, ctypes.byref(count)) == 0
    total = 0
    for node in map(ctypes.c_void_p, nodes):
        kind, params = ctypes.c_int(), KernelNode()
        assert driver.cuGraphNodeGetType(node, ctypes.byref(kind)) == 0
        if kind.value == 0:                               # a kernel
            assert driver.cuGraphKernelNodeGetParams_v2(node, ctypes.byref(params)) == 0
            total += params.grid[0] * params.grid[1] * params.grid[2]
    return total


def test_a_long_prompt_among_many_short_requests():
    """Beyond the workspace's bound, turns are many chunks deep: requests without rows do not cost their CTAs for every chunk of the longest one."""
    D, H, HV, lengths = 64, 64, 64, [1] * 100 + [13000] + [1] * 100
    c, state = make(lengths, H, HV, D, BF16, True, device=DEV)
    B, N, total = len(lengths), sum(lengths), -(-max(lengths) // 64)
    work = torch.empty(pp.prefill_workspace_bytes(c["mixed_qkv"], state, starts(lengths).to(DEV), max(lengths)), dtype=torch.uint8, device=DEV)
    places = work.numel() / (H * 16384 + HV * 32768)
    assert places < N // 64 + B                           # it does not hold every chunk at once
    out, final = run(c, state, lengths, HV, D)
    for i in (0, 100, 200):
        rows = slice(sum(lengths[:i]), sum(lengths[:i + 1]))
        part = {k: v[rows] if k in ("mixed_qkv", "a", "b") else v for k, v in c.items()}
        alone = run(part, state[i:i + 1], lengths[i:i + 1], HV, D)
        if lengths[i] > 1:
            assert torch.equal(out[rows], alone[0]) and torch.equal(final[i:i + 1], alone[1])
        else:                                             # alone, a token goes by itself
            assert (final[i] - alone[1][0]).norm() <= 2 ** -18 * alone[1].norm()
    graph, start = torch.cuda.CUDAGraph(keep_graph=True), starts(lengths).to(DEV)
    with torch.cuda.graph(graph):
        pp.gated_delta_rule_packed_prefill(**c, out=out, final_state=final, initial_state=state, query_start=start, max_query_len=max(lengths),
                                           use_qk_l2norm_in_kernel=True, workspace=work)
    # what does not depend on the state takes a CTA for four chunks of every request and head, as many as the longest one has; the chains two a head
    # and request in every turn
    assert ctas_of(graph) <= 2 * HV * B * -(-total // 4)
