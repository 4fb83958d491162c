"""Tracers see torch's operators and no launch: what they record of the expert layers and of the product for serving is the Python
function, or the call is refused.  The launches are left out, so that no device is needed."""
import warnings

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from triton_int8_b200 import kernels as K
from triton_int8_b200 import linear, moe

BF16 = torch.bfloat16
IDS, POS, SRC = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
X, W, WQ, WS, OFFSETS = torch.ones(4, 16, dtype=BF16), torch.ones(4, 2), torch.zeros(1, 8, 16, dtype=torch.int8), torch.ones(1, 8), SRC[:2]
CALLS = {
    "_SortFn": (lambda x: moe.sort_tokens(x, IDS, 3)[0], X),
    "_CombineFn": (lambda r: moe.combine(r, W, POS, SRC), X.repeat(2, 1)),
    "TokenLinearFn": (lambda x: linear.linear_w8a8(x, WQ[0], WS[0]), X),
    "TokenLinearFn experts": (lambda x: moe.expert_linear(x, WQ, WS, OFFSETS), X),
}


@pytest.fixture(autouse=True)
def no_launches(monkeypatch):
    """Host code as it is, but for results that come from memory that no torch operator has written."""
    class Leaves:
        sort_tokens = combine = token_linear = linear = staticmethod(lambda *a: None)

    def empty(*shape):
        assert all(type(n) is int for n in shape)   # sizes in a recorded function are no traced tensors
        return torch.empty(shape, dtype=BF16)
    monkeypatch.setattr(K, "host", lambda: Leaves)
    monkeypatch.setattr(K, "sort_tokens", lambda x, ids, E, align: (empty(ids.numel(), x.shape[1]), OFFSETS.clone(), POS.clone(), SRC.clone()))
    monkeypatch.setattr(K, "combine", lambda rows, w, pos: empty(pos.shape[0], rows.shape[1]))
    monkeypatch.setattr(K, "token_linear", lambda x, wq, ws, offsets, bias, dt: empty(x.shape[0], wq.shape[1]))


@pytest.mark.parametrize("name", CALLS)
def test_a_trace_records_the_function(name):
    f, x = CALLS[name]
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        graph = str(torch.jit.trace(f, x, check_trace=False).graph)
    assert "^" + name.split()[0] in graph, graph


@pytest.mark.parametrize("name", CALLS)
def test_make_fx_is_refused(name):
    f, x = CALLS[name]
    with torch.no_grad(), pytest.raises(RuntimeError, match="make_fx"):
        make_fx(f)(x)


def test_only_frozen_experts_are_traced():
    """The sizes of the segments would be constants of the trace."""
    layer = moe.Int8MoE(128, 128, experts=3, top_k=2).eval()
    with torch.no_grad(), warnings.catch_warnings(), pytest.raises(RuntimeError, match="frozen"):
        warnings.simplefilter("ignore")
        torch.jit.trace(layer, torch.ones(4, 128, dtype=BF16), check_trace=False)
