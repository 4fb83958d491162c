"""Dual tensors: the expert layers and the product for serving have no forward-mode derivative and say so.  It is looked at
ahead of everything else, so that no device is needed here."""
import pytest
import torch
from torch.autograd import forward_ad

from triton_int8_b200 import linear, moe

BF16 = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def built():
    from triton_int8_b200 import build
    build.build()


def _dual(*shape, dtype=BF16):
    return forward_ad.make_dual(torch.ones(shape, dtype=dtype), torch.ones(shape, dtype=dtype))


IDS, POS, SRC = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
X, W, WQ, WS, OFFSETS = torch.ones(4, 16, dtype=BF16), torch.ones(4, 2), torch.zeros(1, 8, 16, dtype=torch.int8), torch.ones(1, 8), SRC[:2]
CALLS = {
    "sort_tokens x": lambda: moe.sort_tokens(_dual(4, 16), IDS, 3),
    "combine rows": lambda: moe.combine(_dual(8, 16), W, POS, SRC),
    "combine weights": lambda: moe.combine(X.repeat(2, 1), _dual(4, 2, dtype=torch.float32), POS, SRC),
    "expert_linear rows": lambda: moe.expert_linear(_dual(4, 16), WQ, WS, OFFSETS),
    "expert_linear scales": lambda: moe.expert_linear(X, WQ, _dual(1, 8, dtype=torch.float32), OFFSETS),
    "expert_linear bias": lambda: moe.expert_linear(X, WQ, WS, OFFSETS, _dual(1, 8)),
    "linear_w8a8 x": lambda: linear.linear_w8a8(_dual(4, 16), WQ[0], WS[0]),
    "linear_w8a8 scales": lambda: linear.linear_w8a8(X, WQ[0], _dual(8, dtype=torch.float32)),
    "linear_w8a8 bias": lambda: linear.linear_w8a8(X, WQ[0], WS[0], _dual(8)),
    "a frozen layer": lambda: linear.Int8FrozenLinear(WQ[0], WS[0])(_dual(4, 16)),
}


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_refused(call, grad):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
        CALLS[call]()


def test_tensors_without_a_tangent_pass_inside_a_level():
    with forward_ad.dual_level():
        _dual(2)   # somebody else's
        with pytest.raises(ValueError, match="CUDA"):
            moe.sort_tokens(X, IDS, 3)
        with pytest.raises(ValueError, match="CUDA"):
            linear.linear_w8a8(X, WQ[0], WS[0])


@pytest.mark.parametrize("name", ["sort", "combine"])
def test_a_tangent_of_the_incoming_gradient_is_refused(name):
    class Ctx:
        saved_tensors = (POS,) if name == "sort" else (X.repeat(2, 1), W, POS, SRC)
        needs_input_grad = (True, True, False, False)
    node = moe._SortFn if name == "sort" else moe._CombineFn
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        node.backward(Ctx, _dual(8, 16) if name == "sort" else _dual(4, 16))
