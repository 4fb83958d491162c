"""Views whose sign is kept beside their memory, as the imaginary part of a conjugate has it: one element is contiguous as it is."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("T,H", [(1, 1), (4, 3)])
def test_sort_combine_and_their_gradients(T, H):
    from triton_int8_b200 import moe
    g = torch.Generator(device=DEV).manual_seed(0)
    view = lambda *s: torch.randn(s, dtype=torch.complex64, device=DEV, generator=g).conj().imag  # noqa: E731
    x, w, dy, ids = view(T, H), view(T, 1), view(T, H), torch.zeros(T, 1, dtype=torch.int64, device=DEV)
    assert x.is_neg()
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 1)
    assert torch.equal(rows, x.clone())
    r = view(T, H)
    assert torch.equal(moe.combine(r, w, pos, src), w.clone() * r.clone())
    a = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(moe.sort_tokens(a, ids, 1)[0], a, dy)[0], dy.clone())
    a, b = r.clone().requires_grad_(), w.clone().requires_grad_()
    da, db = torch.autograd.grad(moe.combine(a, b, pos, src), (a, b), dy)
    terms = a.detach().double() * dy.clone().double()
    assert torch.equal(da, (w * dy).clone())   # a path of at most H products and the additions between threads, each off by 2^-24
    assert ((db.double() - terms.sum(1, keepdim=True)).abs() <= (H + 16) * 2.0 ** -24 * terms.abs().sum(1, keepdim=True)).all()
