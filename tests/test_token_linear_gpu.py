"""linear_w8a8 and expert_linear: integers and scales are fixed, so fp32 results are compared bit for bit with a plain form that
quantizes by the same steps in 32 bits and sums in 64-bit integers; bf16 ones are those rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import I8LError, double_channel, linear, moe
    from triton_int8_b200 import kernels as K

BF16, F32 = torch.bfloat16, torch.float32


def _plain(x, wq, ws, bias):
    """fp32 [R, N] on the CPU for one matrix."""
    xf = x.cpu().float()
    amax = xf.abs().amax(-1, keepdim=True).clamp_min(1e-4)
    q = torch.floor(xf * (torch.reciprocal(amax) * 127.0) + 0.5)
    acc = torch.zeros(x.shape[0], wq.shape[0], dtype=torch.float64)   # exact: below 2^31
    acc += q.double() @ wq.cpu().double().t()
    y = acc.float() * (amax / 127.0) * ws.cpu()
    return y if bias is None else y + bias.cpu().float()


def _weights(g, *shape):
    wq = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)
    return wq.to(DEV), (torch.rand(shape[:-1], generator=g) * 1e-3 + 1e-4).to(DEV)


def _rows(g, R, Kd):
    x = torch.randn(R, Kd, generator=g) * torch.rand(R, 1, generator=g).mul(4).exp()
    return x.to(BF16).to(DEV)


DENSE = [   # rows, N, K: one row to many, sizes that fill no tile
    (1, 8, 16), (1, 4096, 4096), (2, 1000, 2048), (3, 40, 48), (5, 136, 4112), (8, 256, 11008), (9, 264, 144), (16, 128, 128), (17, 1408, 1040),
    (33, 128, 112), (63, 520, 512), (64, 64, 64), (65, 72, 2064), (127, 384, 256), (128, 128, 128), (129, 136, 144), (255, 1000, 272), (257, 264, 400),
    (300, 128, 16), (1000, 2176, 1408), (2048, 512, 1024), (1, 64, 131072), (4, 72, 81936), (40, 72, 40976),
    (20, 200, 2064), (50, 1288, 2304), (100, 3016, 3200), (64, 1024, 4096), (65, 1024, 4096), (129, 2048, 3088),   # K shared by a cluster
    (700, 2200, 272), (333, 9480, 48), (970, 4768, 144), (439, 9688, 80), (900, 3208, 400), (1537, 2056, 112),   # tiles of 96, 112, 144, 160, 192, 208
]


@pytest.mark.parametrize("R,N,Kd", DENSE)
@pytest.mark.parametrize("with_bias", [False, True])
def test_dense(R, N, Kd, with_bias):
    g = torch.Generator().manual_seed(R + N + Kd)
    x, (wq, ws) = _rows(g, R, Kd), _weights(g, N, Kd)
    bias = torch.randn(N, generator=g).to(BF16).to(DEV) if with_bias else None
    ref = _plain(x, wq, ws, bias)
    assert torch.equal(linear.linear_w8a8(x, wq, ws, bias, out_dtype=F32).cpu(), ref)
    assert torch.equal(linear.linear_w8a8(x, wq, ws, bias).cpu(), ref.to(BF16))
    K.check_status(DEV)


GROUPED = [   # rows of each expert, rows behind the last one, N, K
    ([1], 0, 64, 128), ([0, 1, 0, 1], 0, 4096, 1024), ([0, 0, 0], 3, 64, 48), ([2, 0, 5, 1], 2, 136, 208), ([8], 1, 96, 256), ([9, 0, 7], 0, 128, 144),
    ([64, 1, 0, 65, 16], 5, 264, 400), ([100] * 12, 0, 72, 128), ([0, 0, 700], 130, 128, 256), ([255, 256, 257, 1], 0, 320, 384),
    ([128, 384, 0, 128], 128, 256, 512), ([513, 31, 2000], 77, 1000, 272), ([1] * 60, 4, 40, 64), ([5, 0, 30, 1], 2, 136, 2080), ([9, 64, 0, 70], 3, 264, 4112), ([0, 33], 0, 3000, 3200), ([0] * 1000 + [3, 0, 40] + [0] * 21, 1, 24, 112),
]


@pytest.mark.parametrize("sizes,behind,N,Kd", GROUPED)
@pytest.mark.parametrize("with_bias", [False, True])
def test_experts(sizes, behind, N, Kd, with_bias):
    g = torch.Generator().manual_seed(len(sizes) + sum(sizes) + N)
    E, R = len(sizes), sum(sizes) + behind
    x, (wq, ws) = _rows(g, R, Kd), _weights(g, E, N, Kd)
    bias = torch.randn(E, N, generator=g).to(BF16).to(DEV) if with_bias else None
    offsets = torch.tensor([0] + sizes).cumsum(0).int().to(DEV)
    ref = torch.zeros(R, N)
    for e, (a, b) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
        if b > a:
            ref[a:b] = _plain(x[a:b], wq[e], ws[e], None if bias is None else bias[e])
    x[sum(sizes):] = float("nan")   # rows of no expert come out zero whatever they hold
    assert torch.equal(moe.expert_linear(x, wq, ws, offsets, bias, out_dtype=F32).cpu(), ref)
    assert torch.equal(moe.expert_linear(x, wq, ws, offsets, bias).cpu(), ref.to(BF16))
    K.check_status(DEV)


def test_rows_in_front_of_the_first_expert_and_offsets_out_of_range():
    g = torch.Generator().manual_seed(3)
    for R in (6, 300):
        x, (wq, ws) = _rows(g, R, 64), _weights(g, 3, 40, 64)
        got = moe.expert_linear(x, wq, ws, torch.tensor([2, 2, 5, 5], dtype=torch.int32, device=DEV), out_dtype=F32).cpu()
        ref = torch.zeros(R, 40)
        ref[2:5] = _plain(x[2:5], wq[1], ws[1], None)
        assert torch.equal(got, ref)
        # what reaches out of the rows is cut off
        got = moe.expert_linear(x, wq, ws, torch.tensor([-9, 1, R + 100, 2 ** 31 - 1], dtype=torch.int32, device=DEV), out_dtype=F32).cpu()
        ref = torch.cat([_plain(x[:1], wq[0], ws[0], None), _plain(x[1:], wq[1], ws[1], None)])
        assert torch.equal(got, ref)
    K.check_status(DEV)


@pytest.mark.parametrize("R", [5, 200, 1000])
def test_offsets_that_decrease_touch_nothing_else(R):
    """Overlapping segments: y is undefined, what lies around it is not touched, and the next call is right."""
    g = torch.Generator().manual_seed(R)
    E, N = 64, 136
    x, (wq, ws) = _rows(g, R, 64), _weights(g, E, N, 64)
    offsets = torch.tensor([0, R] * (E // 2) + [0], dtype=torch.int32, device=DEV)
    y = moe.expert_linear(x, wq, ws, offsets)
    torch.cuda.synchronize()
    assert y.shape == (R, N)
    offsets = torch.tensor([0] + [R] * E, dtype=torch.int32, device=DEV)
    assert torch.equal(moe.expert_linear(x, wq, ws, offsets, out_dtype=F32).cpu(), _plain(x, wq[0], ws[0], None))
    K.check_status(DEV)


@pytest.mark.parametrize("M,N,Kd", [(128, 256, 384), (256, 128, 1024), (512, 640, 128)])
def test_bit_equal_to_double_channel(M, N, Kd):
    g = torch.Generator().manual_seed(M)
    a, b = _rows(g, M, Kd), _rows(g, N, Kd)
    wq, ws = moe.quantize_experts(b)
    assert torch.equal(linear.linear_w8a8(a, wq, ws), double_channel.fwd_32(a[None], b, hadamard=None)[0])


def test_largest_sums_do_not_overflow():
    """131072 products of 127 and -128: the sum of largest size."""
    Kd = 131072
    for R in (1, 40):
        x = torch.ones(R, Kd, dtype=BF16, device=DEV)
        wq = torch.full((8, Kd), -128, dtype=torch.int8, device=DEV)
        y = linear.linear_w8a8(x, wq, torch.ones(8, device=DEV), out_dtype=F32)
        assert torch.equal(y.cpu(), _plain(x, wq, torch.ones(8), None))


def test_rows_that_are_zero_tiny_or_not_finite():
    """The floor of a row's maximum is 1e-4; an infinity makes its own row NaN, as the double_channel quantizer has it; NaN counts as zero."""
    for R in (4, 40):
        x = torch.randn(R, 128, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
        wq, ws = _weights(torch.Generator().manual_seed(2), 16, 128)
        x[0], x[1] = 0, x[1] * 1e-8
        ref = _plain(x, wq, ws, None)
        x[2, 5], x[3, 7] = float("inf"), float("nan")
        y = linear.linear_w8a8(x, wq, ws, out_dtype=F32).cpu()
        assert torch.equal(y[:2], ref[:2]) and torch.equal(y[4:], ref[4:]) and y[2].isnan().all()
        x[3, 7] = 0
        assert torch.equal(y[3:4], _plain(x[3:4], wq, ws, None))


def test_leading_dimensions_layouts_and_alignment():
    g = torch.Generator().manual_seed(4)
    x, (wq, ws) = _rows(g, 12, 64), _weights(g, 48, 64)
    bias = torch.randn(48, generator=g).to(BF16).to(DEV)
    want = linear.linear_w8a8(x, wq, ws, bias)
    assert torch.equal(linear.linear_w8a8(x.view(2, 6, 64), wq, ws, bias), want.view(2, 6, 48))
    assert torch.equal(linear.linear_w8a8(x[0], wq, ws, bias), want[0])
    assert linear.linear_w8a8(x[:0], wq, ws, bias).shape == (0, 48)
    off = lambda t: torch.cat([t.view(-1)[:1], t.reshape(-1)])[1:].view(t.shape)   # noqa: E731  off the 16-byte boundary
    assert off(x).data_ptr() % 16 and off(wq).data_ptr() % 16
    for form in (off, lambda t: t if t.dim() < 2 else t.t().contiguous().t()):
        assert torch.equal(linear.linear_w8a8(form(x), form(wq), form(ws), form(bias)), want)
    one = moe.expert_linear(x, wq[None], ws[None], torch.tensor([0, 12], dtype=torch.int32, device=DEV), bias[None])
    assert torch.equal(one, want)


def test_refusals():
    x, wq, ws = torch.zeros(4, 64, dtype=BF16, device=DEV), torch.zeros(2, 16, 64, dtype=torch.int8, device=DEV), torch.ones(2, 16, device=DEV)
    offsets = torch.zeros(3, dtype=torch.int32, device=DEV)
    for bad in (dict(rows=x.half()), dict(rows=x[:, :32]), dict(wq=wq.int()), dict(wq=wq[0]), dict(ws=ws.half()), dict(ws=ws[:1]), dict(ws=ws[:, :8]),
                dict(offsets=offsets.long()), dict(offsets=offsets[:2]), dict(offsets=offsets.cpu()), dict(bias=torch.zeros(16, dtype=BF16, device=DEV)),
                dict(bias=torch.zeros(2, 16, device=DEV)), dict(out_dtype=torch.float16), dict(wq=wq.cpu())):
        with pytest.raises((TypeError, ValueError)):
            moe.expert_linear(**dict(dict(rows=x, wq=wq, ws=ws, offsets=offsets), **bad))
    with pytest.raises(I8LError, match="SHAPE"):
        linear.linear_w8a8(x[:, :56].contiguous(), wq[0, :, :56], ws[0])
    with pytest.raises(I8LError, match="SHAPE"):
        linear.linear_w8a8(x, wq[0, :12], ws[0, :12])
    with pytest.raises(RuntimeError, match="no gradient"):
        linear.linear_w8a8(x.requires_grad_(), wq[0], ws[0])
    with torch.no_grad():
        linear.linear_w8a8(x, wq[0], ws[0])


def test_streams_and_graphs_that_live_together():
    """Two captured calls of different sizes, replayed in turn on new values: neither uses what the other keeps."""
    g = torch.Generator().manual_seed(9)
    graphs = []
    for R, E in ((3, 4), (200, 4)):
        x, (wq, ws) = _rows(g, R, 256), _weights(g, E, 136, 256)
        offsets = torch.tensor([0, R // 3, R // 3, R - 1, R], dtype=torch.int32, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            moe.expert_linear(x, wq, ws, offsets)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = moe.expert_linear(x, wq, ws, offsets)
        graphs.append((graph, x, wq, ws, offsets, y))
    for turn in range(3):
        for graph, x, wq, ws, offsets, y in graphs:
            x.copy_(_rows(g, *x.shape))
            offsets.copy_(offsets.roll(0) if turn == 0 else torch.tensor([0, 1, x.shape[0] - turn, x.shape[0] - turn, x.shape[0]], device=DEV))
        for graph, *_ in graphs:
            graph.replay()
        for graph, x, wq, ws, offsets, y in graphs:
            assert torch.equal(y, moe.expert_linear(x, wq, ws, offsets))
    K.check_status(DEV)


def test_elements_beyond_32_bits():
    """Weights of more than 2^31 bytes and an output of more than 2^31 elements."""
    E, N, Kd = 9, 16384, 16384
    wq = torch.empty(E, N, Kd, dtype=torch.int8, device=DEV)
    wq.zero_()
    wq[:, :, 0] = 1
    wq[E - 1, N - 8:, :16] = torch.arange(16, dtype=torch.int8, device=DEV)
    ws = torch.ones(E, N, device=DEV)
    for R in (2, 40):
        x = torch.ones(R, Kd, dtype=BF16, device=DEV)
        offsets = torch.tensor([0] * E + [R], dtype=torch.int32, device=DEV)
        y = moe.expert_linear(x, wq, ws, offsets, out_dtype=F32)
        assert torch.equal(y[:, -9:].cpu(), _plain(x, wq[-1, -9:], ws[-1, -9:], None))
    del wq
    R, N = 140000, 16384
    x = (torch.arange(R, device=DEV) % 255 - 127).to(BF16)[:, None].expand(R, 16).contiguous()
    wq, ws = _weights(torch.Generator().manual_seed(1), N, 16)
    y = linear.linear_w8a8(x, wq, ws)
    pick = torch.tensor([0, 1, 65535, 131071, 131072, 139998, 139999], device=DEV)
    assert y.numel() > 2 ** 31 and torch.equal(y[pick].cpu(), _plain(x[pick], wq, ws, None).to(BF16))


@pytest.mark.parametrize("R,E,N,Kd", [(200, 1, 2048, 512), (3000, 4, 1000, 272), (3000, 4, 20000, 272), (20, 1, 200, 2064), (50, 1, 1288, 2304),
                                      (100, 2, 1504, 3200), (60, 2, 40, 9008)])
def test_wait_that_runs_out_and_the_next_call(R, E, N, Kd):
    """A withheld load: the kernel returns, the status word says so, the next call is right (see test_timeout_gpu.py)."""
    from triton_int8_b200 import _lib as L
    lib = L.load()
    g = torch.Generator().manual_seed(11)
    x, (wq, ws) = _rows(g, R, Kd), _weights(g, E, N, Kd)
    offsets = torch.tensor([R * e // E for e in range(E + 1)], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert lib.i8l_test_set_wait_limit(256, 1) == 0
    try:
        K.token_linear(x, wq, ws, offsets, status=status)
        torch.cuda.synchronize()
    finally:
        assert lib.i8l_test_set_wait_limit(0, 0) == 0
    assert status.item() == L.TIMEOUT
    status.zero_()
    y = K.token_linear(x, wq, ws, offsets, out_dtype=F32, status=status)
    assert status.item() == 0
    ref = torch.cat([_plain(x[a:b], wq[e], ws[e], None) for e, (a, b) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:]))])
    assert torch.equal(y.cpu(), ref)
