"""A frozen layer computes the same behind casts of the model that it is part of."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cast", [lambda m: m.float(), lambda m: m.half(), lambda m: m.half().to(torch.bfloat16), lambda m: m.cpu().float().cuda()])
def test_the_result_is_unchanged(cast):
    from triton_int8_b200 import linear
    torch.manual_seed(0)
    lin = linear.Int8Linear(256, 128, bias=True, device="cuda")
    with torch.no_grad():
        lin.bias.normal_()
    model = torch.nn.Sequential(lin.freeze())
    x = torch.randn(6, 256, device="cuda").to(torch.bfloat16)
    y = model(x)
    assert torch.equal(cast(model)(x), y)
