"""Gradients of the expert layers where hooks on saved tensors give back other tensors than were saved: laid out otherwise they count for what they
hold, of another type, shape or device they are refused."""
import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import kernels as K
    from triton_int8_b200 import moe


@pytest.fixture(params=["native", "python"], autouse=True)
def path(request, monkeypatch):
    if request.param == "python":
        class Leaves:
            sort_tokens = combine = token_linear = staticmethod(lambda *a: None)
        monkeypatch.setattr(K, "host", lambda: Leaves)


def _grads(hooks, H=24):
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(40, H, device=DEV, generator=g).requires_grad_()
    w, ids = torch.rand(40, 3, device=DEV, generator=g).requires_grad_(), torch.randint(-1, 5, (40, 3), device=DEV, generator=g)
    dy = torch.randn(40, H, device=DEV, generator=g)
    with saved_tensors_hooks(*hooks):
        rows, offsets, pos, src = moe.sort_tokens(x, ids, 5, align=4)
        y = moe.combine(rows, w, pos, src)
    return torch.autograd.grad(y, (x, w), dy)


def _other_layout(t):
    if t.dim() == 2:
        return t.t().contiguous().t()
    return torch.stack([t, t], 1)[:, 0]


@pytest.mark.parametrize("H", [24, 25])
@pytest.mark.parametrize("pack,unpack", [(lambda t: t.cpu(), lambda t: t.to(DEV)), (lambda t: t, _other_layout), (lambda t: t, lambda t: t.clone())])
def test_other_places_and_layouts(pack, unpack, H):
    same = (lambda t: t, lambda t: t)
    assert all(torch.equal(a, b) for a, b in zip(_grads((pack, unpack), H), _grads(same, H)))


@pytest.mark.parametrize("unpack", [lambda t: t.cpu(), lambda t: t.double(), lambda t: t[:-1]])
def test_what_does_not_fit_is_refused(unpack):
    with pytest.raises((RuntimeError, ValueError, TypeError)):
        _grads((lambda t: t, unpack))


def test_recomputation():
    from torch.utils.checkpoint import checkpoint
    x = torch.randn(300, 16, device=DEV).requires_grad_()
    w, ids = torch.rand(300, 2, device=DEV).requires_grad_(), torch.randint(0, 5, (300, 2), device=DEV)

    def f(x, w):
        rows, offsets, pos, src = moe.sort_tokens(x.sin(), ids, 5)
        return moe.combine(rows.cos(), w, pos, src)
    want = torch.autograd.grad(f(x, w).square().sum(), (x, w))
    got = torch.autograd.grad(checkpoint(f, x, w, use_reentrant=False).square().sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
