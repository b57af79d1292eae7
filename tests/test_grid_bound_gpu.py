"""``max_ctas`` bounds every kernel that a decode variant launches: the grids are read from a captured graph."""

import ctypes as C

import pytest
import torch

import test_decode_modes_gpu as modes
import test_shared_prefix_gpu as prefix
from _serving import Paged

pytestmark = pytest.mark.gpu


class _KernelNode(C.Structure):
    _fields_ = [("func", C.c_void_p), ("grid", C.c_uint * 3), ("block", C.c_uint * 3), ("shared", C.c_uint), ("params", C.c_void_p),
                ("extra", C.c_void_p), ("room", C.c_void_p * 4)]


def _grids(call):
    """CTAs of each kernel that `call` launches."""
    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = call()  # noqa: F841
    cuda, raw, n, kind = C.CDLL("libcuda.so.1"), C.c_void_p(graph.raw_cuda_graph()), C.c_size_t(), C.c_int()
    assert cuda.cuGraphGetNodes(raw, None, C.byref(n)) == 0
    nodes, got = (C.c_void_p * n.value)(), []
    assert cuda.cuGraphGetNodes(raw, nodes, C.byref(n)) == 0
    for node in nodes:
        assert cuda.cuGraphNodeGetType(C.c_void_p(node), C.byref(kind)) == 0
        if kind.value == 0:
            p = _KernelNode()
            assert cuda.cuGraphKernelNodeGetParams(C.c_void_p(node), C.byref(p)) == 0
            got.append(p.grid[0] * p.grid[1] * p.grid[2])
    return got


@pytest.mark.parametrize("bound", [1, 5, 40, 0])
@pytest.mark.parametrize("op", ["window", "weights", "prefix"])
def test_every_grid_is_bounded(op, bound):
    from cleave_b200 import ops

    if op == "prefix":
        c = prefix.Case(1500, [300] * 70, 16, 4, 64, 16, torch.bfloat16, seed=1)
        q, k, v, *rest = c.args()
        pre = c.pre_ids.to(torch.int32).cuda()
        call = lambda: ops.gqa_paged_decode_shared_prefix(q, k, v, pre, 1500, *rest, max_ctas=bound)  # noqa: E731
    else:
        c = Paged([3000, 500, 2000, 70], 16, 4, 64, 16, torch.bfloat16, seed=1)
        args, sums = c.args(), torch.zeros(4, 4, 3000, device="cuda")
        call = ((lambda: ops.gqa_paged_decode_window(*args, 1000, 4, max_ctas=bound)) if op == "window" else
                (lambda: ops.gqa_paged_decode_weights(*args, sums, max_ctas=bound)))
    got = _grids(call)
    assert len(got) >= (1 if op == "window" else 2)
    if bound:
        assert max(got) <= bound, got
    else:
        assert max(got) > 40  # the cases are large enough for the bounds to matter


@pytest.mark.parametrize("bound", [1, 5, 40])
def test_bounded_prefix(bound):
    prefix.Case(700, [0, 1, 300, 64] + [5] * 40, 16, 4, 64, 16, torch.float16, seed=2).check(max_ctas=bound)
    prefix.Case(700, [0, 1, 300], 8, 2, 128, 64, torch.bfloat16, seed=3).check(max_ctas=bound)


@pytest.mark.parametrize("bound", [1, 2, 5, 40])
@pytest.mark.parametrize("max_len", [5000, 300])
def test_bounded_weights(max_len, bound):
    modes._check_weights(Paged([3000, 1, 300, 0, 2049], 8, 2, 64, 16, torch.bfloat16, seed=4), max_len, steps=2, max_ctas=bound)
