"""Traced modules compute what the modules do, for other inputs and other numbers of tokens than those of the trace."""
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import linear, moe

BF16 = torch.bfloat16


def _trace(f, *x):
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        return torch.jit.trace(f, x, check_trace=False)


def _poison():
    """Memory that the allocator hands out next holds no earlier result."""
    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 22):
        torch.full((n,), float("nan"), device=DEV)


@pytest.mark.parametrize("bias", [True, False])
def test_a_frozen_linear(bias):
    torch.manual_seed(0)
    frozen = linear.Int8Linear(256, 384, bias=bias, device=DEV).freeze()
    traced = _trace(frozen, torch.randn(5, 256, device=DEV).to(BF16))
    for shape in ((5, 256), (1, 256), (300, 256)):
        x = torch.randn(shape, device=DEV).to(BF16)
        with torch.no_grad():
            want = frozen(x)
            _poison()
            assert torch.equal(traced(x), want)


def test_frozen_experts():
    torch.manual_seed(1)
    layer = moe.Int8MoE(256, 384, experts=5, top_k=2, device=DEV).eval().freeze()
    traced = _trace(layer, torch.randn(7, 256, device=DEV).to(BF16))
    for tokens in (7, 1, 333):
        x = torch.randn(tokens, 256, device=DEV).to(BF16)
        with torch.no_grad():
            want = layer(x)
            _poison()
            assert torch.equal(traced(x), want)


def test_sort_and_combine():
    def f(x, ids, w):
        rows, offsets, pos, src = moe.sort_tokens(x, ids, 6, align=4)
        return moe.combine(rows, w, pos, src), offsets, rows

    def inputs(T):
        return torch.randn(T, 72, device=DEV), torch.randint(-1, 6, (T, 3), device=DEV), torch.rand(T, 3, device=DEV)
    traced = _trace(f, *inputs(9))
    for T in (9, 1, 2500):
        args = inputs(T)
        with torch.no_grad():
            want = f(*args)
            _poison()
            assert all(torch.equal(a, b) for a, b in zip(traced(*args), want))
