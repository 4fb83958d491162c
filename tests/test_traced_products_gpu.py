"""No graph holds the allocation of a result without the launch that fills it: the functions refuse to be traced, Int8Linear is a node of a trace."""
import warnings

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import block_channel, double_channel, fused
    from triton_int8_b200.linear import Int8Config, Int8Linear

BF16 = torch.bfloat16


def _trace(f, x):
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        return torch.jit.trace(f, x, check_trace=False)


CALLS = {
    "block_channel.fwd_32": lambda x, w: block_channel.fwd_32(x, w),
    "block_channel.bwd_33": lambda x, w: block_channel.bwd_33(x, w[None]),
    "quantizer": lambda x, w: block_channel.triton_per_block_quant(x)[0],
    "double_channel.fwd_32": lambda x, w: double_channel.fwd_32(x, w),
    "fused.fwd_32": lambda x, w: fused.fwd_32(x, w),
    "fused, one kernel": lambda x, w: fused.fwd_32(x, w, single_kernel=True),
}


@pytest.mark.parametrize("name", CALLS)
def test_functions_refuse_tracers(name):
    x, w = torch.randn(1, 128, 256, device=DEV).to(BF16), torch.randn(256, 256, device=DEV).to(BF16)
    f = lambda t: CALLS[name](t, w)  # noqa: E731
    with pytest.raises(RuntimeError, match="jit.trace"):
        _trace(f, x)
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(f)(x)
    assert torch.isfinite(f(x).float()).all()   # and run as before


@pytest.mark.parametrize("cfg", [{}, dict(scaling="double_channel"), dict(scaling="double_channel", hadamard=-1)])
def test_a_traced_int8_linear(cfg):
    torch.manual_seed(0)
    lin = Int8Linear(256, 384, device=DEV, config=Int8Config(**cfg))
    with torch.no_grad():
        lin.bias.normal_()
    traced = _trace(lin, torch.randn(128, 256, device=DEV).to(BF16))
    for shape in ((128, 256), (384, 256)):
        x = torch.randn(shape, device=DEV).to(BF16)
        with torch.no_grad():
            want = lin(x)
            torch.full((1 << 20,), float("nan"), device=DEV)
            assert torch.equal(traced(x), want)
    with torch.no_grad(), pytest.raises(RuntimeError, match="make_fx"):
        make_fx(lin)(torch.randn(128, 256, device=DEV).to(BF16))
