"""sort_tokens and combine with their gradients against plain loops and 64-bit sums."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import kernels as K
    from triton_int8_b200 import moe

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    """The native host path, and the Python one that takes what it leaves."""
    if request.param == "python":
        class Leaves:
            sort_tokens = combine = token_linear = staticmethod(lambda *a: None)
        monkeypatch.setattr(K, "host", lambda: Leaves)


def _plain_layout(ids, experts, align, rows):
    """offsets, pos, src by a loop over the choices."""
    flat = ids.reshape(-1).tolist()
    count = [0] * experts
    place = []
    for e in flat:
        place.append(count[e] if 0 <= e < experts else -1)
        if 0 <= e < experts:
            count[e] += 1
    offsets = [0]
    for c in count:
        offsets.append(offsets[-1] + -(-c // align) * align)
    pos = [offsets[e] + at if at >= 0 else -1 for e, at in zip(flat, place)]
    src = [-1] * rows
    for i, r in enumerate(pos):
        if r >= 0:
            src[r] = i
    return (torch.tensor(offsets, dtype=torch.int32), torch.tensor(pos, dtype=torch.int32).view(ids.shape), torch.tensor(src, dtype=torch.int32))


def _half_step(dtype, value):
    """A rounding to dtype is off by at most half a step: eps / 2 of the value, and half the smallest subnormal near zero."""
    info = torch.finfo(dtype)
    return info.eps / 2 * value.abs() + info.smallest_normal * info.eps / 2


def _values(g, shape, dtype):
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


CASES = [   # tokens, columns, choices, experts, align, type, ids, share dropped
    (0, 8, 2, 4, 1, BF16, torch.int64, 0.0),
    (0, 8, 2, 4, 16, F32, torch.int32, 0.0),
    (1, 1, 1, 1, 1, BF16, torch.int32, 0.0),
    (1, 4096, 2, 8, 1, BF16, torch.int64, 0.0),
    (3, 7, 2, 5, 1, F16, torch.int32, 0.3),
    (17, 129, 3, 7, 128, F32, torch.int64, 0.5),
    (128, 256, 8, 60, 1, BF16, torch.int64, 0.0),      # 1024 choices: one launch
    (205, 264, 5, 64, 16, F16, torch.int64, 0.2),      # 1025: three
    (1024, 72, 1, 1024, 3, BF16, torch.int32, 0.1),
    (1025, 40, 1, 1024, 2, BF16, torch.int64, 0.0),
    (40, 24, 64, 33, 1, F32, torch.int32, 0.0),
    (1999, 1405, 4, 8, 128, BF16, torch.int64, 0.9),
    (5000, 8, 7, 2, 1, F16, torch.int32, 0.0),
    (70000, 8, 1, 100, 1, BF16, torch.int64, 0.5),
    (2048, 40000, 1, 3, 1, F16, torch.int32, 0.0),     # rows longer than a block's passes
]


def _ids(g, T, k, E, dtype, drop):
    ids = torch.randint(0, E, (T, k), generator=g)
    return torch.where(torch.rand(T, k, generator=g) < drop, torch.where(ids % 2 == 0, -1, E + ids), ids).to(dtype)


@pytest.mark.parametrize("T,H,k,E,align,dtype,idt,drop", CASES)
def test_sort_and_its_gradient(path, T, H, k, E, align, dtype, idt, drop):
    g = torch.Generator().manual_seed(T + H)
    x, ids = _values(g, (T, H), dtype).requires_grad_(), _ids(g, T, k, E, idt, drop)
    rows, offsets, pos, src = moe.sort_tokens(x, ids.to(DEV), E, align)
    R = K.sorted_rows(T, k, E, align)
    ref_offsets, ref_pos, ref_src = _plain_layout(ids, E, align, R)
    assert torch.equal(offsets.cpu(), ref_offsets) and torch.equal(pos.cpu(), ref_pos) and torch.equal(src.cpu(), ref_src)
    expect = torch.zeros((R, H), dtype=dtype)
    live = ref_src >= 0
    expect[live] = x.detach().cpu()[ref_src[live].long() // k]
    assert torch.equal(rows.detach().cpu(), expect)
    drows = _values(g, (R, H), dtype)
    (dx,) = torch.autograd.grad(rows, x, drows)
    d = drows.cpu().double()
    ref = torch.zeros(T, H, dtype=torch.float64).index_add_(0, ref_src[live].long() // k, d[live])
    size = torch.zeros(T, H, dtype=torch.float64).index_add_(0, ref_src[live].long() // k, d[live].abs())
    # at most k - 1 additions in 32 bits, each off by 2^-24 of a partial sum, then one rounding
    err = (dx.cpu().double() - ref).abs()
    assert (err <= (k - 1) * 2.0 ** -24 * size * 1.01 + _half_step(dtype, size)).all(), float(err.max())
    with torch.no_grad():   # the same without a graph
        again = moe.sort_tokens(x, ids.to(DEV), E, align)
    assert all(torch.equal(a, b) for a, b in zip(again, (rows, offsets, pos, src)))


@pytest.mark.parametrize("T,H,k,E,align,dtype,idt,drop", CASES)
@pytest.mark.parametrize("wide_weights", [True, False])
def test_combine_and_its_gradients(path, T, H, k, E, align, dtype, idt, drop, wide_weights):
    g = torch.Generator().manual_seed(T + 3 * H)
    R = K.sorted_rows(T, k, E, align)
    _, pos, src = _plain_layout(_ids(g, T, k, E, idt, drop), E, align, R)
    rows = _values(g, (R, H), dtype)
    rows[src.to(DEV) < 0] = float("nan")             # rows of no choice are not looked at
    weights = torch.rand(T, k, generator=g).to(F32 if wide_weights else dtype)
    weights[pos < 0] = float("inf")                  # nor are the weights of dropped choices
    weights = weights.to(DEV)
    rows.requires_grad_(), weights.requires_grad_()
    y = moe.combine(rows, weights, pos.to(DEV), src.to(DEV))
    dy = _values(g, (T, H), dtype)
    drows, dweights = torch.autograd.grad(y, (rows, weights), dy)

    live = src >= 0
    at = src[live].long()
    r64, w64, dy64 = rows.detach().cpu().double()[live], weights.detach().cpu().double().view(-1)[at][:, None], dy.cpu().double()[at // k]
    zero = torch.zeros(T, H, dtype=torch.float64)
    ref, size = zero.index_add(0, at // k, w64 * r64), zero.index_add(0, at // k, (w64 * r64).abs())
    err = (y.detach().cpu().double() - ref).abs()
    # k fused multiply-additions in 32 bits, one rounding
    bound = k * 2.0 ** -24 * size * 1.01
    assert (err <= bound + _half_step(dtype, ref.abs() + bound)).all(), float(err.max())

    ref = torch.zeros(R, H, dtype=torch.float64)
    ref[live] = w64 * dy64
    err = (drows.cpu().double() - ref).abs()          # one product in 32 bits, one rounding
    assert (err <= 2.0 ** -24 * ref.abs() * 1.01 + _half_step(dtype, ref * (1 + 2.0 ** -24))).all(), float(err.max())
    assert (drows[(src < 0).to(DEV)] == 0).all()

    ref, size = torch.zeros(T * k, dtype=torch.float64), torch.zeros(T * k, dtype=torch.float64)
    ref[at], size[at] = (r64 * dy64).sum(-1), (r64 * dy64).abs().sum(-1)
    err = (dweights.cpu().double().view(-1) - ref).abs()
    # a thread adds up to H fused products, then the threads' sums are added: no path of more than H + 16 additions
    bound = (H + 16) * 2.0 ** -24 * size * 1.01
    assert (err <= bound + _half_step(weights.dtype, ref.abs() + bound)).all(), float(err.max())
    assert (dweights[(pos < 0).to(DEV)] == 0).all()


def test_gradients_against_differences(path):
    """y is linear in x and in the weights: a difference over a whole step is the derivative, up to the roundings of 32 bits."""
    g = torch.Generator().manual_seed(5)
    T, H, k, E = 37, 100, 3, 5
    x, w = _values(g, (T, H), F32).requires_grad_(), torch.rand(T, k, generator=g).to(DEV).requires_grad_()
    ids = _ids(g, T, k, E, torch.int64, 0.2).to(DEV)
    scale = _values(g, (1, H), F32)

    def f(x, w):
        rows, offsets, pos, src = moe.sort_tokens(x, ids, E, align=4)
        return moe.combine(rows * scale, w, pos, src)
    dy, dx, dw = _values(g, (T, H), F32), _values(g, (T, H), F32), _values(g, (T, k), F32)
    gx, gw = torch.autograd.grad(f(x, w), (x, w), dy)
    with torch.no_grad():
        for grad, step, moved in ((gx, dx, f(x + dx, w) - f(x, w)), (gw, dw, f(x, w + dw) - f(x, w))):
            a, b = float((grad.double() * step.double()).sum()), float((moved.double() * dy.double()).sum())
            # values up to 5 * 5 * 5 * 3, T * H terms with 2^-24 of that each at most; typical terms are 1
            assert abs(a - b) <= 2.0 ** -24 * 375 * T * H, (a, b)


def test_only_the_gradients_that_are_wanted(path):
    g = torch.Generator().manual_seed(6)
    x, ids = _values(g, (6, 16), BF16), torch.randint(0, 3, (6, 2), generator=g).to(DEV)
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 3)
    assert not rows.requires_grad
    w = torch.rand(6, 2, device=DEV)
    both = [t.clone().requires_grad_() for t in (rows, w)]
    want = torch.autograd.grad(moe.combine(*both, pos, src).sum(), both)
    for i in (0, 1):
        t = [rows, w]
        t[i] = t[i].clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(moe.combine(*t, pos, src).sum(), t[i])[0], want[i])
    with torch.no_grad():
        assert not moe.combine(*both, pos, src).requires_grad


def test_a_second_gradient_is_refused(path):
    x, ids = torch.randn(6, 16, device=DEV).requires_grad_(), torch.randint(0, 3, (6, 2), device=DEV)
    w = torch.rand(6, 2, device=DEV).requires_grad_()
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 3)
    (dx,) = torch.autograd.grad(rows.square().sum(), x, create_graph=True)   # its incoming gradient depends on x
    with pytest.raises(RuntimeError, match="twice"):
        dx.sum().backward()
    y = moe.combine(rows.detach().requires_grad_(), w, pos, src)
    (dw,) = torch.autograd.grad(y.sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dw.sum().backward()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_layouts_that_are_not_contiguous_or_aligned(dtype):
    g = torch.Generator().manual_seed(7)
    T, H, k, E = 50, 64, 2, 4
    flat = _values(g, (T * H + 8,), dtype)
    base = flat[:T * H].view(T, H)
    ids = torch.randint(0, E, (T, k), generator=g).to(DEV)
    shifted = flat.clone()[1:]                                   # off the 16-byte boundary by an element
    shifted[:T * H] = flat[:T * H]
    shifted = shifted[:T * H].view(T, H)
    forms = [base.t().contiguous().t(), torch.cat([base, base], 1)[:, :H], shifted, base[:, None].expand(T, 1, H)[:, 0]]
    want = moe.sort_tokens(base, ids, E)
    assert shifted.data_ptr() % 16
    for form in forms:
        assert all(torch.equal(a, b) for a, b in zip(moe.sort_tokens(form, ids.t().contiguous().t(), E), want))
    rows, offsets, pos, src = want
    w = torch.rand(T, k, device=DEV)
    y = moe.combine(rows, w, pos, src)
    big = torch.empty(rows.numel() + 1, dtype=dtype, device=DEV)
    big[1:] = rows.view(-1)
    for r in (rows.t().contiguous().t(), big[1:].view(rows.shape)):
        r = r.detach().requires_grad_()
        y2 = moe.combine(r, w.t().contiguous().t(), pos.t().contiguous().t(), src)
        assert torch.equal(y, y2)
        (a,) = torch.autograd.grad(y2.sum(), r)                  # the gradient of a sum is an expanded one
        (b,) = torch.autograd.grad(moe.combine(rows.requires_grad_(), w, pos, src), rows, torch.ones_like(y))
        assert torch.equal(a, b)


def test_the_same_expert_twice_and_positions_out_of_range():
    x = torch.arange(8, device=DEV, dtype=F32).view(2, 4)
    rows, offsets, pos, src = moe.sort_tokens(x, torch.tensor([[1, 1], [1, 0]], device=DEV), 2)
    assert offsets.tolist() == [0, 1, 4] and pos.tolist() == [[1, 2], [3, 0]] and src.tolist() == [3, 0, 1, 2]
    w = torch.tensor([[1., 2.], [3., 4.]], device=DEV)
    assert torch.equal(moe.combine(rows, w, pos, src), torch.stack([3 * x[0], 7 * x[1]]))
    wild = torch.tensor([[1, 4], [-7, 2 ** 31 - 1]], device=DEV, dtype=torch.int32)   # rows there are: 4
    r = rows.clone().requires_grad_()
    y = moe.combine(r, w, wild, src)
    assert torch.equal(y, torch.stack([rows[1], torch.zeros(4, device=DEV)]))
    (d,) = torch.autograd.grad(y.sum(), r)
    assert torch.equal(d[1], torch.ones(4, device=DEV)) and torch.isfinite(d[1]).all()


def test_infinities_and_nan_pass_through():
    x = torch.tensor([[float("inf"), 1.0], [float("nan"), -2.0]], device=DEV, dtype=BF16)
    rows, offsets, pos, src = moe.sort_tokens(x, torch.tensor([[1], [0]], device=DEV), 2)
    y = moe.combine(rows, torch.ones(2, 1, device=DEV), pos, src)
    assert torch.equal(torch.nan_to_num(y, 7.0, 9.0), torch.nan_to_num(x, 7.0, 9.0))


def test_streams_and_graphs(path):
    """On a stream of its own, captured and replayed on new values and new choices, the backward pass in the graph too."""
    g = torch.Generator().manual_seed(8)
    for T in (4, 900):   # one launch, three
        H, k, E = 136, 2, 6
        x, w = _values(g, (T, H), BF16).requires_grad_(), torch.rand(T, k, generator=g).to(DEV).requires_grad_()
        ids, dy = torch.randint(0, E, (T, k), generator=g).to(DEV), _values(g, (T, H), BF16)

        def step():
            rows, offsets, pos, src = moe.sort_tokens(x, ids, E, align=8)
            y = moe.combine(rows, w, pos, src)
            return (y.detach(), offsets, *torch.autograd.grad(y, (x, w), dy))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        for seed in range(2):
            with torch.no_grad():
                x.copy_(_values(g, (T, H), BF16))
                w.copy_(torch.rand(T, k, generator=g).to(DEV))
                ids.copy_(torch.randint(0, E, (T, k), generator=g).to(DEV))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in captured]
            want = step()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_wrappers_refuse_shapes_and_types(path):
    x, ids = torch.zeros(4, 8, dtype=BF16, device=DEV), torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    for bad in (dict(x=x.double()), dict(x=x.int()), dict(x=x[0]), dict(x=x[None]), dict(ids=ids.short()), dict(ids=ids.float()), dict(ids=ids[:3]),
                dict(ids=ids[:, 0]), dict(experts=0), dict(align=0), dict(ids=ids.cpu())):
        a = dict(x=x, ids=ids, experts=4, align=1)
        a.update(bad)
        with pytest.raises((TypeError, ValueError)):
            moe.sort_tokens(**a)
    from triton_int8_b200 import I8LError
    for bad in (dict(experts=1025), dict(ids=torch.zeros(4, 65, dtype=torch.int64, device=DEV)), dict(align=65537)):
        with pytest.raises(I8LError, match="SHAPE"):
            moe.sort_tokens(**dict(dict(x=x, ids=ids, experts=4), **bad))
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 4)
    w = torch.ones(4, 2, device=DEV)
    for bad in (dict(rows=rows.double()), dict(weights=w.half()), dict(weights=w[:3]), dict(pos=pos.long()), dict(pos=pos.view(-1)), dict(pos=pos.cpu()),
                dict(src=src[1:], weights=w.clone().requires_grad_())):
        a = dict(rows=rows, weights=w, pos=pos, src=src)
        a.update(bad)
        with pytest.raises((TypeError, ValueError)):
            moe.combine(**a)


def test_rows_beyond_32_bit_offsets():
    """More than 2^31 elements in the rows: addresses are 64-bit."""
    T, H, k = 33000, 33024, 2
    x = torch.empty(T, H, dtype=BF16, device=DEV)
    x[:] = (torch.arange(T, device=DEV) % 251).to(BF16)[:, None]
    ids = torch.stack([torch.zeros(T, dtype=torch.int32), torch.ones(T, dtype=torch.int32)], 1).to(DEV)
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 2)
    assert rows.numel() > 2 ** 31 and offsets.tolist() == [0, T, 2 * T]
    assert torch.equal(rows[-1], x[-1]) and torch.equal(rows[T], x[0]) and torch.equal(rows[T + 1:][::997], x[1:][::997])
    y = moe.combine(rows, torch.ones(T, k, device=DEV), pos, src)
    assert torch.equal(y[::997], 2 * x[::997])
    drows, dweights = K.combine_backward(rows, torch.full((T, k), 2.0, device=DEV), pos, src, x)
    assert torch.equal(drows[T:][::997], 2 * x[::997])
    ref = (x[::997].double() ** 2).sum(-1)
    assert ((dweights[::997, 1].double() - ref).abs() <= (H + 16) * 2.0 ** -24 * ref).all()


def test_transforms_are_refused():
    """The kernels cannot see through a batched tensor: an error, not numbers."""
    x, ids = torch.randn(6, 16, device=DEV).requires_grad_(), torch.randint(0, 3, (6, 2), device=DEV)
    w = torch.rand(6, 2, device=DEV).requires_grad_()
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 3)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(rows, x, torch.randn(3, *rows.shape, device=DEV), is_grads_batched=True, retain_graph=True)
    y = moe.combine(rows.detach().requires_grad_(), w, pos, src)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, w, torch.randn(3, *y.shape, device=DEV), is_grads_batched=True)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda r: moe.combine(r, w.detach(), pos, src))(torch.randn(2, *rows.shape, device=DEV))


def test_changed_inputs_and_a_second_pass_are_noticed(path):
    x, ids = torch.randn(6, 16, device=DEV).requires_grad_(), torch.randint(0, 3, (6, 2), device=DEV)
    w = torch.rand(6, 2, device=DEV).requires_grad_()
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 3)
    rows.sum().backward(retain_graph=True)
    rows.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 4.0))
    r = rows.detach().requires_grad_()
    y = moe.combine(r, w, pos, src)
    with torch.no_grad():
        r.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_calls_from_several_threads_on_streams_of_their_own():
    import threading

    from triton_int8_b200.moe import expert_linear
    q, s = K.quant_row(torch.randn(8 * 256, 512, device=DEV).to(BF16), 3)
    q, s, bad = q.view(8, 256, 512), s.view(8, 256), []

    def work(seed):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            g = torch.Generator(device=DEV).manual_seed(seed)
            for T in (3, 7, 40, 700) * 3:
                x = torch.randn(T, 512, device=DEV, generator=g).to(BF16).requires_grad_()
                offsets = torch.linspace(0, T, 9, device=DEV).int()
                ids = torch.randint(0, 8, (T, 2), device=DEV, generator=g)
                stream.synchronize()   # the weights, and what the generators made
                same = torch.equal(expert_linear(x.detach(), q, s, offsets), expert_linear(x.detach(), q, s, offsets))
                rows, _, pos, src = moe.sort_tokens(x, ids, 8)
                y = moe.combine(rows, torch.ones(T, 2, device=DEV), pos, src)
                (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
                if not same or not torch.equal(y, (2 * x.detach().float()).to(BF16)) or not torch.equal(dx, torch.full_like(dx, 2.0)):
                    bad.append((seed, T))
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    K.check_status(DEV)


def test_capture_beside_a_living_eager_graph_does_not_end_the_process(tmp_path):
    """torch cannot capture a backward pass whose leaves belong to an eager graph on another stream: an exception, in a child process here."""
    import os
    import subprocess
    import sys
    script = tmp_path / "child.py"
    script.write_text("""
import torch
from triton_int8_b200 import moe
x = torch.randn(900, 136, device="cuda").requires_grad_()
w, ids = torch.rand(900, 2, device="cuda").requires_grad_(), torch.randint(0, 6, (900, 2), device="cuda")
def forward():
    rows, offsets, pos, src = moe.sort_tokens(x, ids, 6)
    return moe.combine(rows, w, pos, src)
eager, dy = forward(), torch.randn(900, 136, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph):
        torch.autograd.grad(forward(), (x, w), dy)
except RuntimeError as e:
    print("raised", type(e).__name__)
dx, dw = torch.autograd.grad(eager, (x, w), dy)   # the eager graph still is what it was
assert torch.isfinite(dx).all() and torch.isfinite(dw).all()
print("alive")
""")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, str(script)], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "alive" in done.stdout, done.stdout + done.stderr[-2000:]
