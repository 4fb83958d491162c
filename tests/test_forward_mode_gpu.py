"""Dual tensors on the device: refused by both host paths, on the way back too."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import kernels as K
    from triton_int8_b200 import linear, moe


@pytest.fixture(params=["native", "python"], autouse=True)
def path(request, monkeypatch):
    if request.param == "python":
        class Leaves:
            sort_tokens = combine = token_linear = staticmethod(lambda *a: None)
        monkeypatch.setattr(K, "host", lambda: Leaves)


def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def test_duals_are_refused():
    x, ids = torch.randn(6, 16, device=DEV), torch.randint(0, 3, (6, 2), device=DEV)
    w = torch.rand(6, 2, device=DEV)
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 3)
    frozen = linear.Int8Linear(128, 128, device=DEV).freeze()
    with forward_ad.dual_level():
        for call in (lambda: moe.sort_tokens(_dual(x), ids, 3), lambda: moe.combine(_dual(rows), w, pos, src),
                     lambda: moe.combine(rows, _dual(w), pos, src), lambda: frozen(_dual(torch.ones(5, 128, device=DEV, dtype=torch.bfloat16)))):
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        moe.sort_tokens(x, ids, 3)   # without a tangent


def test_a_dual_gradient_on_the_way_back_is_refused():
    """Forward over reverse: the tangent of what comes in would be lost."""
    x, ids = torch.randn(6, 16, device=DEV).requires_grad_(), torch.randint(0, 3, (6, 2), device=DEV)
    w = torch.rand(6, 2, device=DEV).requires_grad_()
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 3)
    y = moe.combine(rows.detach().requires_grad_(), w, pos, src)
    for out, leaf in ((rows, x), (y, w)):
        with forward_ad.dual_level(), pytest.raises((NotImplementedError, RuntimeError)):
            torch.autograd.grad(out, leaf, _dual(torch.ones_like(out)), retain_graph=True)
        assert torch.isfinite(torch.autograd.grad(out, leaf, torch.ones_like(out))[0]).all()
