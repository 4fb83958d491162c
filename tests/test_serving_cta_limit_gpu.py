"""kernels.cta_limit holds for the product for serving, with few rows too: the launches of a captured call, and its results."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import kernels as K
    from triton_int8_b200 import moe


class _Node(ctypes.Structure):   # CUDA_KERNEL_NODE_PARAMS_v2
    _fields_ = [("func", ctypes.c_void_p), ("grid", ctypes.c_uint * 3), ("block", ctypes.c_uint * 3), ("smem", ctypes.c_uint),
                ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p), ("kern", ctypes.c_void_p), ("ctx", ctypes.c_void_p)]


def _launches(call):
    """Blocks of each kernel that the call launches, in no particular order."""
    cuda = ctypes.CDLL("libcuda.so.1")
    call()   # outside of the capture first: status word, attributes
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert cuda.cuGraphGetNodes(raw, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert cuda.cuGraphGetNodes(raw, nodes, ctypes.byref(count)) == 0
    grids = []
    for node in nodes:
        kind, params = ctypes.c_int(-1), _Node()
        assert cuda.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        if kind.value == 0:   # a kernel
            assert cuda.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), ctypes.byref(params)) == 0
            grids.append(params.grid[0] * params.grid[1] * params.grid[2])
    return grids


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("experts", [1, 6])
def test_few_rows(rows, experts):
    g = torch.Generator(device=DEV).manual_seed(rows)
    wq = torch.randint(-127, 128, (experts, 296, 512), generator=g, device=DEV, dtype=torch.int8)
    ws, x = torch.rand(experts, 296, generator=g, device=DEV), torch.randn(rows, 512, generator=g, device=DEV).to(torch.bfloat16)
    offsets = torch.linspace(0, rows, experts + 1, device=DEV).int()
    call = lambda: moe.expert_linear(x, wq, ws, offsets)  # noqa: E731
    want, free = call(), _launches(call)
    assert len(free) == 1
    for limit in (1, 5, 40):
        with K.cta_limit(limit):
            assert torch.equal(call(), want)
            assert _launches(call)[0] == min(limit, free[0])
    assert _launches(call) == free   # the limit has ended
    with K.cta_limit(100000):        # more than there are SMs
        assert _launches(call) == free
