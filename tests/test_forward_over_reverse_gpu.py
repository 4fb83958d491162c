"""Int8Linear's backward pass on a dual gradient: the products have no forward-mode derivative and say so, the bias gradient is a sum and has one."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import kernels as K
    from triton_int8_b200.linear import Int8Config, Int8Linear


@pytest.mark.parametrize("path", ["native", "python"])
@pytest.mark.parametrize("cfg", [{}, dict(scaling="double_channel", hadamard=-1)])
def test_a_dual_gradient(path, cfg, monkeypatch):
    if path == "python":
        class Leaves:
            linear = quant_gemm = staticmethod(lambda *a: None)
        monkeypatch.setattr(K, "host", lambda: Leaves)
    torch.manual_seed(0)
    lin = Int8Linear(256, 128, bias=True, device=DEV, config=Int8Config(**cfg))
    x, dy, t = (torch.randn(128, n, device=DEV).to(torch.bfloat16) for n in (256, 128, 128))
    y = lin(x.requires_grad_())
    for of in (x, lin.weight):
        with forward_ad.dual_level(), pytest.raises((NotImplementedError, RuntimeError)):
            torch.autograd.grad(y, of, forward_ad.make_dual(dy, t), retain_graph=True)
    with forward_ad.dual_level():
        lin.requires_grad_(False).bias.requires_grad_()
        (db,) = torch.autograd.grad(lin(x.detach()), lin.bias, forward_ad.make_dual(dy, t))
        got = forward_ad.unpack_dual(db)
        assert got.tangent is not None and torch.equal(got.tangent, t.sum(0))
