"""Backward passes that run under a mode (a counter of operations, a default device) which the forward passes did not see."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import moe


class Sees(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("mode", [Sees, lambda: torch.device("cuda"), lambda: torch.device("cpu"),
                                  lambda: torch.overrides.BaseTorchFunctionMode()])
@pytest.mark.parametrize("H", [16, 17])
def test_gradients_are_the_same(mode, H):
    g = torch.Generator(device=DEV).manual_seed(1)
    x, w = torch.randn(50, H, device=DEV, generator=g).requires_grad_(), torch.rand(50, 2, device=DEV, generator=g).requires_grad_()
    ids, dy = torch.randint(-1, 4, (50, 2), device=DEV, generator=g), torch.randn(50, H, device=DEV, generator=g)
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 4, align=8)
    y = moe.combine(rows, w, pos, src)
    want = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    with mode():
        got = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
        whole = moe.combine(moe.sort_tokens(x, ids, 4, align=8)[0], w, pos, src)   # and both passes under it
        both = torch.autograd.grad(whole, (x, w), dy)
    assert torch.equal(whole, y)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, both))
