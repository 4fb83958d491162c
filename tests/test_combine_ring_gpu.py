"""combine, its gradients and that of sort_tokens at the sizes of the kernel for many tokens (rows of whole 16 bytes, above 512 of them; 2048 tokens
forward, 1024 backward, up to 32 choices) and on both sides of its limits, against 64-bit sums."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import kernels as K
    from triton_int8_b200 import moe

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _half_step(dtype, value):
    """A rounding to dtype is off by at most half a step: eps / 2 of the value, and half the smallest subnormal near zero."""
    info = torch.finfo(dtype)
    return info.eps / 2 * value.abs() + info.smallest_normal * info.eps / 2


def _within(got, ref, sums, roundings, dtype):
    """`roundings` operations in 32 bits, each off by 2^-24 of at most the sum of the sizes of all terms, then one rounding to dtype."""
    bound = roundings * 2.0 ** -24 * sums * 1.01
    err = (got.double() - ref).abs()
    assert (err <= bound + _half_step(dtype, ref.abs() + bound)).all(), float(err.max())


CASES = [   # tokens, columns, choices, experts, align, type, weights in 32 bits, share dropped
    (2049, 264, 3, 8, 16, BF16, True, 0.3),       # half of the second stage, a third of a segment
    (2500, 1032, 8, 60, 1, F32, True, 0.25),      # three segments of 512 columns
    (3001, 520, 5, 7, 128, F16, False, 0.5),
    (2048, 1032, 1, 4, 64, BF16, False, 0.9),     # most rows are cleared
    (2051, 264, 32, 40, 1, BF16, True, 0.2),      # a choice a lane
    (2051, 264, 33, 40, 1, BF16, True, 0.2),      # one more
    (2047, 264, 2, 8, 1, BF16, True, 0.3), (1024, 264, 4, 8, 8, F16, True, 0.3), (1023, 264, 4, 8, 8, F16, True, 0.3),
    (2100, 256, 3, 8, 1, BF16, True, 0.3),        # 512 bytes
    (5000, 132, 7, 16, 1, F32, True, 1.0),        # all dropped
    (2400, 2056, 2, 3, 1, BF16, True, 0.0),
]


def _make(T, H, k, E, align, dtype, wide, drop):
    g = torch.Generator(device=DEV).manual_seed(T + H + k)
    ids = torch.randint(0, E, (T, k), device=DEV, generator=g)
    ids = torch.where(torch.rand(T, k, device=DEV, generator=g) < drop, torch.where(ids % 2 == 0, -1, E + ids), ids)
    x = torch.randn(T, H, device=DEV, generator=g).to(dtype)
    rows, offsets, pos, src = moe.sort_tokens(x, ids, E, align)
    live = src >= 0
    rows = torch.randn(rows.shape, device=DEV, generator=g).to(dtype)
    rows[~live] = float("nan")                    # rows of no choice are not looked at
    weights = torch.rand(T, k, device=DEV, generator=g).to(F32 if wide else dtype)
    weights[pos < 0] = float("inf")               # nor are the weights of dropped choices
    return x, ids, rows, weights, pos, src, live, torch.randn(T, H, device=DEV, generator=g).to(dtype)


@pytest.mark.parametrize("T,H,k,E,align,dtype,wide,drop", CASES)
def test_combine_and_its_gradients(T, H, k, E, align, dtype, wide, drop):
    x, ids, rows, weights, pos, src, live, dy = _make(T, H, k, E, align, dtype, wide, drop)
    rows.requires_grad_(), weights.requires_grad_()
    y = moe.combine(rows, weights, pos, src)
    drows, dweights = torch.autograd.grad(y, (rows, weights), dy, retain_graph=True)
    at = src[live].long()
    r64, w64, dy64 = rows.detach()[live].double(), weights.detach().view(-1)[at].double()[:, None], dy.double()[at // k]
    zero = torch.zeros(T, H, dtype=torch.float64, device=DEV)
    _within(y.detach(), zero.index_add(0, at // k, w64 * r64), zero.index_add(0, at // k, (w64 * r64).abs()), k, dtype)
    ref = torch.zeros(drows.shape, dtype=torch.float64, device=DEV)
    ref[live] = w64 * dy64
    _within(drows, ref, ref.abs(), 1, dtype)
    assert (drows[~live] == 0).all()
    ref, size = torch.zeros(2, T * k, dtype=torch.float64, device=DEV)
    ref[at], size[at] = (r64 * dy64).sum(-1), (r64 * dy64).abs().sum(-1)
    _within(dweights.view(-1), ref, size, H + 16, weights.dtype)   # a path of at most H products and the additions between threads
    assert (dweights[pos < 0] == 0).all()
    # one gradient alone is the same
    assert torch.equal(moe.combine(rows, weights.detach(), pos, src), y)
    for of, want in ((rows, drows), (weights, dweights)):
        args = [rows.detach(), weights.detach(), pos, src]
        args[0 if of is rows else 1] = of
        assert torch.equal(torch.autograd.grad(moe.combine(*args), of, dy)[0], want)


@pytest.mark.parametrize("T,H,k,E,align,dtype,wide,drop", CASES)
def test_gradient_of_the_sort(T, H, k, E, align, dtype, wide, drop):
    x, ids, drows, _, pos, src, live, _ = _make(T, H, k, E, align, dtype, wide, drop)
    rows = moe.sort_tokens(x.requires_grad_(), ids, E, align)[0]
    assert torch.equal(rows.detach()[live], x.detach()[src[live].long() // k]) and not rows[~live].any()
    (dx,) = torch.autograd.grad(rows, x, drows)
    d, zero, token = drows[live].double(), torch.zeros(T, H, dtype=torch.float64, device=DEV), src[live].long() // k
    _within(dx, zero.index_add(0, token, d), zero.index_add(0, token, d.abs()), k, dtype)


def test_the_kernel_for_many_tokens_in_a_graph():
    """Captured and replayed on other values and positions, gradients too."""
    case = (2300, 520, 3, 6, 8, BF16, True, 0.3)
    x, ids, rows, weights, pos, src, live, dy = _make(*case)
    rows, weights = rows.nan_to_num().requires_grad_(), weights.nan_to_num(posinf=1.0).requires_grad_()

    def step():
        y = moe.combine(rows, weights, pos, src)
        return (y.detach(), *torch.autograd.grad(y, (rows, weights), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(2):
        g = torch.Generator(device=DEV).manual_seed(seed)
        _, _, p, s = moe.sort_tokens(x, torch.randint(-2, 6, ids.shape, device=DEV, generator=g), 6, 8)
        with torch.no_grad():
            pos.copy_(p), src.copy_(s), dy.normal_(generator=g), weights.uniform_(generator=g), rows.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    K.check_status(DEV)
