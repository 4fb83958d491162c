"""Casts of a frozen layer: weights, scales and bias stay what the product reads, with their values."""
import pytest
import torch

from triton_int8_b200.linear import Int8FrozenLinear


@pytest.mark.parametrize("cast", [lambda m: m.float(), lambda m: m.half(), lambda m: m.double(), lambda m: m.to(torch.float16),
                                  lambda m: torch.nn.Sequential(m).half()[0], lambda m: m.bfloat16().half().float()])
def test_casts_keep_every_value(cast):
    g = torch.Generator().manual_seed(0)
    q, scale = torch.randint(-127, 128, (16, 32), generator=g, dtype=torch.int8), torch.rand(16, generator=g)
    bias = torch.randn(16, generator=g).to(torch.bfloat16)
    bias[:3] = torch.tensor([1e30, -1e-30, 3e5]).to(torch.bfloat16)   # outside of what fp16 holds
    frozen = cast(Int8FrozenLinear(q.clone(), scale.clone(), bias.clone()))
    for name, want in (("weight_q", q), ("weight_scale", scale), ("bias", bias)):
        got = frozen.state_dict()[name]
        assert got.dtype == want.dtype and torch.equal(got, want), name
        assert got is not None and getattr(frozen, name).data_ptr() == got.data_ptr()


def test_a_bias_of_another_type_is_cast():
    frozen = Int8FrozenLinear(torch.zeros(16, 32, dtype=torch.int8), torch.ones(16), torch.ones(16)).to(torch.bfloat16)
    assert frozen.bias.dtype == torch.bfloat16
    assert Int8FrozenLinear(torch.zeros(16, 32, dtype=torch.int8), torch.ones(16)).half().bias is None


def test_moving_to_another_device_moves_all():
    frozen = Int8FrozenLinear(torch.zeros(16, 32, dtype=torch.int8), torch.ones(16), torch.ones(16, dtype=torch.bfloat16))
    frozen = frozen.to(device="meta", dtype=torch.float16)
    assert {t.device.type for t in frozen.buffers()} == {"meta"}
    assert frozen.bias.dtype == torch.bfloat16 and frozen.weight_scale.dtype == torch.float32
