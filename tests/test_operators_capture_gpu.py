"""What the differentiable operators put into a captured graph, and their replays."""

from __future__ import annotations

import ctypes

import pytest
import torch

from verification.computation import operators as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
MEMSET = 2  # hipGraphNodeTypeMemset


def _kinds(graph):
    """The types of a captured graph's nodes, from the runtime that torch itself has loaded."""
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    hip = ctypes.CDLL(path)
    raw, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    assert hip.hipGraphGetNodes(raw, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert hip.hipGraphGetNodes(raw, nodes, ctypes.byref(count)) == 0
    out = []
    for node in nodes:
        kind = ctypes.c_int(-1)
        assert hip.hipGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        out.append(kind.value)
    return out


@pytest.mark.parametrize("rows", [300, 65536, 65537, 1 << 20])
def test_a_captured_loss_clears_no_memory_by_memset(rows):
    """Such a node has given wrong results on later replays. Replays on new inputs, the eager call
    between them."""
    g = torch.Generator().manual_seed(rows)
    w = torch.randn(50, 16, generator=g).bfloat16().to(DEV)
    t = torch.randint(-1, 50, (rows,), generator=g).to(DEV)
    x = torch.empty(rows, 16, dtype=torch.bfloat16, device=DEV)
    weights = torch.empty(rows, device=DEV)

    def new_inputs():
        x.copy_(torch.randn(rows, 16, generator=g))
        weights.copy_(torch.rand(rows, generator=g) / rows)

    def step():
        leaves = [a.detach().requires_grad_() for a in (x, w, weights)]
        loss = ops.vocab_loss(leaves[0], leaves[1], t, leaves[2])
        return loss.detach(), *torch.autograd.grad(loss, leaves)

    new_inputs()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        held = step()
    assert MEMSET not in _kinds(graph)
    graph.instantiate()
    for _ in range(3):
        new_inputs()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
