"""The expert layer as it is used: routing, sorting, experts and the way back in one module, trained and served, also in a decoder layer."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda"

if torch.cuda.is_available():
    from triton_int8_b200 import linear, moe
    from triton_int8_b200 import kernels as K
    from triton_int8_b200.decoder_layer import DecoderLayer

BF16 = torch.bfloat16


def _rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


def _layer(seed=0, **kw):
    torch.manual_seed(seed)
    return moe.Int8MoE(256, 384, experts=5, top_k=2, device=DEV, **kw)


def _plain(layer, x):
    """fp32 of the same weights and the same choices, token by token over all experts."""
    ids, w = layer.route(x)
    y = torch.zeros(x.shape, device=DEV, dtype=torch.float32)
    xf = x.float()
    for e in range(layer.experts):
        g, u, d = (m[e].weight.float() for m in (layer.gate_proj, layer.up_proj, layer.down_proj))
        part = F.linear(F.silu(F.linear(xf, g)) * F.linear(xf, u), d)
        y = y + part * (w * (ids == e)).sum(-1, keepdim=True)
    return y


@pytest.mark.parametrize("tokens", [1, 3, 128, 333])
def test_training_pass_with_experts_that_are_exact(tokens):
    """bf16 experts (nn.Linear) in place of the INT8 ones: what is left are bf16 roundings, of which there are seven between x and y (three
    linears, silu, product, two products' operands; each at most 2^-8 of its value) and eleven on the way back."""
    layer = _layer(linear=lambda i, o: torch.nn.Linear(i, o, bias=False, device=DEV, dtype=BF16))
    x = torch.randn(tokens, 256, device=DEV).to(BF16).requires_grad_()
    dy = torch.randn(tokens, 256, device=DEV).to(BF16)
    y = layer(x)
    grads = torch.autograd.grad(y, [x, layer.router.weight, *(m.weight for m in layer.gate_proj)], dy, allow_unused=True)
    x2 = x.detach().clone().requires_grad_()
    ref = _plain(layer, x2)
    want = torch.autograd.grad(ref, [x2, layer.router.weight, *(m.weight for m in layer.gate_proj)], dy.float(), allow_unused=True)
    assert _rel(y, ref) <= 7 * 2 ** -8
    for a, b in zip(grads, want):
        if a is None:   # an expert without tokens
            assert b is None or not b.any()
        elif b.any():
            assert _rel(a, b) <= 11 * 2 ** -8


def test_training_pass_runs_and_has_all_gradients():
    layer = _layer()
    x = torch.randn(4, 50, 256, device=DEV).to(BF16).requires_grad_()
    layer(x).sum().backward()
    assert x.grad.shape == x.shape and torch.isfinite(x.grad).all()
    for name, p in layer.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    K.check_status(DEV)


@pytest.mark.parametrize("tokens", [1, 2, 4, 5, 64, 333])
def test_served_pass_is_the_operators_one_after_the_other(tokens):
    layer = _layer(1).eval().freeze()
    x = torch.randn(tokens, 256, device=DEV).to(BF16)
    with torch.no_grad():
        y = layer(x)
        ids, w = layer.route(x)
        out = torch.zeros(tokens, 256, dtype=torch.float32, device=DEV)
        for j in range(layer.top_k):   # every choice for itself through the dense product
            for t in range(tokens):
                e = int(ids[t, j])
                lin = [linear.Int8FrozenLinear.from_linear(m[e]) for m in (layer.gate_proj, layer.up_proj, layer.down_proj)]
                part = lin[2](F.silu(lin[0](x[t:t + 1])) * lin[1](x[t:t + 1]))
                out[t] = torch.addcmul(out[t], w[t, j], part[0].float())
    # the same integers and roundings; the sum over the choices is two fused products in 32 bits, rounded once
    err = (y.float() - out).abs()
    size = out.abs() + 1e-30
    assert (err <= 2.0 ** -8 * size + 4 * 2.0 ** -24 * out.abs().max()).all(), float((err / size).max())
    K.check_status(DEV)


def test_served_pass_against_training_pass_and_fp32():
    layer = _layer(2).eval().freeze()
    x = torch.randn(256, 256, device=DEV).to(BF16)
    with torch.no_grad():
        y, ref = layer(x), _plain(layer, x)
    # int8 operands: a step of amax / 127 is rounded, uniform errors of 1 / sqrt(12) steps against values of amax / 3 at least in rms give
    # 3 / (127 sqrt(12)) = 0.7 % an operand; six operands in three products, none worse than added up
    assert _rel(y, ref) <= 6 * 3 / (127 * 12 ** 0.5) + 7 * 2 ** -8
    assert layer._frozen is not None and layer.train()._frozen is None
    assert layer.eval().freeze()._frozen is not None
    layer.load_state_dict(_layer(3).state_dict())     # other weights: the copy of the old ones goes
    with torch.no_grad():
        assert layer._frozen is None and torch.equal(layer(x), _layer(3).eval()(x))
    assert layer.freeze().to(DEV)._frozen is None
    with pytest.raises(ValueError):
        moe.Int8MoE(128, 128, experts=2, top_k=3, device=DEV)


def test_served_pass_in_a_graph():
    layer = _layer(3).eval().freeze()
    x = torch.randn(5, 256, device=DEV).to(BF16)
    side = torch.cuda.Stream()
    with torch.no_grad():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(x)
        for seed in range(3):
            x.copy_(torch.randn(5, 256, device=DEV))
            graph.replay()
            assert torch.equal(y, layer(x))


def test_frozen_linear():
    torch.manual_seed(4)
    lin = linear.Int8Linear(256, 136 * 128 // 8, bias=True, device=DEV)
    frozen = lin.freeze()
    x = torch.randn(3, 7, 256, device=DEV).to(BF16)
    y = frozen(x)
    q, s = K.quant_row(lin.weight.detach(), 3)
    assert y.shape == (3, 7, lin.out_features) and torch.equal(y, linear.linear_w8a8(x, q, s, lin.bias.detach()))
    assert set(frozen.state_dict()) == {"weight_q", "weight_scale", "bias"}
    with pytest.raises(RuntimeError, match="no gradient"):
        frozen(x.requires_grad_())


def test_decoder_layer_with_experts():
    torch.manual_seed(5)
    layer = DecoderLayer(hidden=256, heads=4, mlp=384, device=DEV, experts=4, top_k=2)
    x = (0.1 * torch.randn(2, 128, 256, device=DEV)).to(BF16).requires_grad_()
    layer(x).sum().backward()
    assert torch.isfinite(x.grad).all() and layer.moe.router.weight.grad is not None
    assert set(layer.linears()) == {"q_proj", "k_proj", "v_proj", "o_proj"}
    layer.eval()
    layer.moe.freeze()
    with torch.no_grad():
        h = layer(x)
    assert torch.isfinite(h).all()
    plain = DecoderLayer(hidden=256, heads=4, mlp=384, device=DEV)
    assert len(plain.linears()) == 7 and plain(x.detach()).shape == x.shape
    K.check_status(DEV)


@pytest.mark.parametrize("where", ["all", "up", "down"])
def test_frozen_experts_keep_their_biases(where):
    """Bit for bit what each expert's frozen linears give on its rows."""
    built = []

    def build(i, o):   # gates first, then ups, then downs
        bias = where == "all" or where == ("gate", "up", "down")[len(built) // 5]
        built.append(torch.nn.Linear(i, o, bias=bias, device=DEV, dtype=BF16))
        return built[-1]

    layer = _layer(7, linear=build).eval().freeze()
    x = torch.randn(37, 256, device=DEV).to(BF16)
    with torch.no_grad():
        ids, weights = layer.route(x)
        rows, offsets, pos, src = moe.sort_tokens(x, ids, 5)
        ends, parts = offsets.tolist(), []
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            gate, up, down = (linear.Int8FrozenLinear.from_linear(m[e]) for m in (layer.gate_proj, layer.up_proj, layer.down_proj))
            if b > a:
                parts.append(down(F.silu(gate(rows[a:b])) * up(rows[a:b])))
        assert torch.equal(layer(x), moe.combine(torch.cat(parts), weights, pos, src))


def test_frozen_linear_keeps_its_scales_when_it_is_cast():
    torch.manual_seed(8)
    frozen = linear.Int8Linear(256, 128, bias=True, device=DEV).freeze()
    x = torch.randn(6, 256, device=DEV).to(BF16)
    y = frozen(x)
    assert torch.equal(frozen.to(BF16)(x), y) and frozen.weight_scale.dtype == torch.float32


def test_combine_checks_src_without_gradients_too():
    rows, offsets, pos, src = moe.sort_tokens(torch.randn(9, 16, device=DEV), torch.zeros(9, 2, dtype=torch.int64, device=DEV), 3)
    weights = torch.ones(9, 2, device=DEV)
    for wrong, error in ((src[:-1], ValueError), (src.long(), TypeError), (src.cpu(), ValueError)):
        with pytest.raises(error):
            moe.combine(rows, weights, pos, wrong)
