"""The single-kernel fused GEMM gives the same bits in every call: a staging slot is refilled only when all of it has been read.  What let a refill in
front of the last reads was a kernel before it that had left the instruction cache empty, so every call here has one."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("batched", [False, True])
def test_every_call_has_the_same_bits(batched):
    from triton_int8_b200 import fused, linear
    from triton_int8_b200 import kernels as K
    g = torch.Generator(device=DEV).manual_seed(0)
    a = torch.randn(2, 256, 512, device=DEV, generator=g).to(torch.bfloat16)
    b = torch.randn((2, 128, 512) if batched else (384, 512), device=DEV, generator=g).to(torch.bfloat16)
    x = torch.randn(3000, 2064, device=DEV, generator=g).to(torch.bfloat16)
    wq = torch.randint(-127, 128, (72, 2064), device=DEV, generator=g, dtype=torch.int8)
    ws = torch.ones(72, device=DEV)
    want, bad = fused.fused_int8_gemm(a, b, out_dtype=torch.float32, exact=True), torch.zeros((), dtype=torch.int64, device=DEV)
    for _ in range(12000):
        linear.linear_w8a8(x, wq, ws)
        bad += (fused.fused_int8_gemm(a, b, out_dtype=torch.float32, exact=True, single_kernel=True) != want).any()
    assert int(bad) == 0
    K.check_status(DEV)
