"""The product for serving around the sizes where the kernels for few rows hand over to the tensor cores: the same bits on both sides."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import kernels as K
    from triton_int8_b200 import linear, moe


def _plain(x, wq, ws, bias):
    """By the steps of the definition in 32 bits, the sum exact."""
    xf = x.cpu().float()
    amax = xf.abs().amax(-1, keepdim=True).clamp_min(1e-4)
    q = torch.floor(xf * (torch.reciprocal(amax) * 127.0) + 0.5)
    y = (q.double() @ wq.cpu().double().t()).float() * (amax / 127.0) * ws.cpu()
    return y if bias is None else y + bias.cpu().float()


def _inputs(R, E, N, Kd):
    g = torch.Generator().manual_seed(R + E + N + Kd)
    x = (torch.randn(R, Kd, generator=g) * torch.rand(R, 1, generator=g).mul(4).exp()).to(torch.bfloat16)
    wq = torch.randint(-127, 128, (E, N, Kd), generator=g, dtype=torch.int8)
    return x.to(DEV), wq.to(DEV), (torch.rand(E, N, generator=g) * 1e-3 + 1e-4).to(DEV), torch.randn(E, N, generator=g).to(torch.bfloat16).to(DEV)


@pytest.mark.parametrize("R,N,Kd", [
    (1, 24, 32768), (1, 24, 32784), (2, 24, 16384), (2, 24, 16400), (3, 40, 8192), (3, 40, 8208), (4, 72, 8192), (4, 72, 8208),
    (3, 5120, 8192), (3, 5128, 8192), (4, 10240, 4096), (4, 10248, 4096), (5, 264, 4096), (5, 264, 4112), (6, 1000, 4080), (7, 40, 3088), (8, 72, 2064),
    (8, 256, 4096), (8, 256, 4112), (5, 6144, 4096), (5, 6152, 4096), (8, 11008, 2048), (8, 16384, 1536), (8, 16392, 1536)])
def test_dense(R, N, Kd):
    x, wq, ws, bias = _inputs(R, 1, N, Kd)
    want = _plain(x, wq[0], ws[0], bias[0])
    assert torch.equal(linear.linear_w8a8(x, wq[0], ws[0], bias[0], out_dtype=torch.float32).cpu(), want)
    assert torch.equal(linear.linear_w8a8(x, wq[0], ws[0], bias[0]).cpu(), want.to(torch.bfloat16))
    K.check_status(DEV)


@pytest.mark.parametrize("sizes,N,Kd", [
    ([1, 1], 72, 16384), ([2, 2], 48, 8192), ([1, 1, 1, 1], 10248, 80), ([1, 2], 4736, 4096), ([1, 2], 5248, 4096), ([3, 2], 3056, 528), ([3, 2], 3088, 528), ([4, 4], 2056, 4096),
    ([1] * 5, 488, 1040), ([1] * 5, 496, 1040), ([0, 1, 0, 2, 1, 1, 0, 1], 336, 2064), ([1] * 8, 192, 4096), ([1] * 8, 200, 4096), ([0, 8, 0], 1360, 304)])
@pytest.mark.parametrize("behind", [0, 1])
def test_experts(sizes, N, Kd, behind):
    E, R = len(sizes), sum(sizes)
    x, wq, ws, bias = _inputs(R + behind, E, N, Kd)
    offsets = torch.tensor([0] + sizes).cumsum(0).int()
    want = torch.zeros(R + behind, N)
    for e, (a, b) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
        if b > a:
            want[a:b] = _plain(x[a:b], wq[e], ws[e], bias[e])
    assert torch.equal(moe.expert_linear(x, wq, ws, offsets.to(DEV), bias, out_dtype=torch.float32).cpu(), want)
    K.check_status(DEV)
