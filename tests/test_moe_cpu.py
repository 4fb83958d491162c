"""The expert layers and the product for serving: what is refused, before any launch.  No device is needed here: what passes the
checks ends in an architecture or CUDA error."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from triton_int8_b200 import _lib, build
    build.build()
    return _lib.load()


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(1 << 16)
    at = ctypes.addressof(buf)
    yield at + (256 - at % 256) % 256
    del buf


NO_DEVICE = (-3, -4)
gone = pytest.mark.skipif(torch.cuda.is_available(), reason="pointers of no device: checks what is refused before a launch")


@gone
@pytest.mark.parametrize("change,code", [
    ({}, NO_DEVICE), (dict(k=0), -1), (dict(k=65), -1), (dict(tokens=-1), -1), (dict(cols=0), -1), (dict(experts=0), -1),
    (dict(experts=1025), -1), (dict(align=0), -1), (dict(align=65537), -1), (dict(rows=7), -1), (dict(align=4), -1), (dict(dtype=3), -6),
    (dict(dtype=-1), -6), (dict(tokens=1 << 30, k=2), -1), (dict(x=None), -6), (dict(ids=None), -6), (dict(out=None), -6),
    (dict(pos=None), -6), (dict(src=None), -6), (dict(offsets=None), -6), (dict(x=1), -2), (dict(out=1), -2), (dict(ids=4), -2),
    (dict(tokens=1000, rows=2000), -6), (dict(tokens=1000, rows=2000, ws=1 << 12), NO_DEVICE), (dict(dtype=2, x=2), -2),
    (dict(tokens=0, rows=0, x=None, ids=None, out=None, pos=None, src=None), NO_DEVICE),
])
def test_sort_tokens_refusals(lib, p, change, code):
    a = dict(x=0, ids=0, tokens=4, cols=8, k=2, experts=4, align=1, dtype=0, rows=8, out=0, offsets=0, pos=0, src=0, ws=0)
    a.update(change)
    at = lambda off: None if off is None else p + off  # noqa: E731
    rc = lib.i8l_sort_tokens(at(a["x"]), at(a["ids"]), 1, a["tokens"], a["cols"], a["k"], a["experts"], a["align"], a["dtype"], a["rows"],
                             at(a["out"]), at(a["offsets"]), at(a["pos"]), at(a["src"]), p, a["ws"], None)
    assert rc in (code if isinstance(code, tuple) else (code,)), lib.i8l_last_error()


@gone
@pytest.mark.parametrize("change,code", [
    ({}, NO_DEVICE), (dict(k=0), -1), (dict(k=65), -1), (dict(cols=0), -1), (dict(dtype=7), -6), (dict(wdtype=1), -6), (dict(wdtype=2), NO_DEVICE),
    (dict(rows=None), -6), (dict(y=None), -6), (dict(pos=None), -6), (dict(rows=1), -2), (dict(y=1), -2), (dict(pos=2), -2), (dict(tokens=0), 0),
    (dict(weights=None), NO_DEVICE), (dict(n_rows=-1), -1), (dict(n_rows=1 << 31), -1),
])
def test_combine_refusals(lib, p, change, code):
    a = dict(rows=0, weights=0, pos=0, n_rows=8, tokens=4, cols=8, k=2, dtype=0, wdtype=0, y=0)
    a.update(change)
    at = lambda off: None if off is None else p + off  # noqa: E731
    rc = lib.i8l_combine(at(a["rows"]), at(a["weights"]), at(a["pos"]), a["n_rows"], a["tokens"], a["cols"], a["k"], a["dtype"], a["wdtype"],
                         at(a["y"]), None)
    assert rc in (code if isinstance(code, tuple) else (code,)), lib.i8l_last_error()
    if set(change) <= {"rows", "pos", "weights", "k", "cols", "dtype", "wdtype", "n_rows"}:
        if change == dict(weights=None):
            code = -6   # ones have no gradient
        if change == dict(pos=2):
            return
        rc = lib.i8l_combine_backward(at(a["rows"]), at(a["weights"]), at(a["pos"]), p, p, a["n_rows"], a["tokens"], a["cols"], a["k"],
                                      a["dtype"], a["wdtype"], p, p, None)
        assert rc in (code if isinstance(code, tuple) else (code,)), lib.i8l_last_error()


@gone
@pytest.mark.parametrize("change,code", [
    ({}, NO_DEVICE), (dict(rows=0), 0), (dict(rows=-1), -1), (dict(N=0), -1), (dict(N=12), -1), (dict(K=24), -1), (dict(K=0), -1),
    (dict(K=131072 + 16), -1), (dict(experts=0), -1), (dict(experts=1025), -1), (dict(offsets=None), -1), (dict(offsets=None, experts=1), NO_DEVICE),
    (dict(flags=1), -6), (dict(flags=4), NO_DEVICE), (dict(x=None), -6), (dict(wq=None), -6), (dict(ws=None), -6), (dict(y=None), -6), (dict(x=8), -2),
    (dict(wq=8), -2), (dict(y=8), -2), (dict(bias=8), -2), (dict(bias=0), NO_DEVICE), (dict(space=0), -6), (dict(work=16), -2), (dict(work=None), -6),
])
def test_token_linear_refusals(lib, p, change, code):
    a = dict(x=0, wq=0, ws=0, offsets=0, bias=None, y=0, rows=9, experts=4, N=16, K=32, flags=0, work=0, space=1 << 14)
    a.update(change)
    at = lambda off: None if off is None else p + off  # noqa: E731
    rc = lib.i8l_token_linear(at(a["x"]), at(a["wq"]), at(a["ws"]), at(a["offsets"]), at(a["bias"]), at(a["y"]), a["rows"], a["experts"], a["N"],
                              a["K"], a["flags"], at(a["work"]), a["space"], None, None)
    assert rc in (code if isinstance(code, tuple) else (code,)), lib.i8l_last_error()


def test_workspace_sizes(lib):
    assert lib.i8l_sort_workspace(512, 2, 8) == 0                      # few choices need none
    assert lib.i8l_sort_workspace(513, 2, 8) == 5 * 8 * 4              # chunks of 256 choices
    assert lib.i8l_sort_workspace(1 << 20, 8, 1024) == 16 * 1024 * 4
    assert lib.i8l_token_linear_workspace(9, 1, 8, 48) == 1280 + 256                 # rows 128 bytes apart
    assert lib.i8l_token_linear_workspace(8, 1, 8, 48) == 0                     # few rows: one launch
    assert lib.i8l_token_linear_workspace(1, 1, 8, 131072) == 131072 + 256      # but long ones
    assert lib.i8l_token_linear_workspace(8, 1, 11008, 4096) == 32768 + 256     # and more than four on many weights
    assert lib.i8l_token_linear_workspace(0, 1, 8, 48) == 0


def test_wrappers_refuse_what_the_kernels_do_not_take():
    from triton_int8_b200 import linear, moe
    x, ids = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        moe.sort_tokens(x, ids, 4)
    with pytest.raises(ValueError, match="CUDA"):
        moe.combine(x, torch.ones(2, 2), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    wq, ws = torch.zeros(16, 8, dtype=torch.int8), torch.ones(16)
    with pytest.raises(ValueError, match="CUDA"):
        linear.linear_w8a8(x, wq, ws)
    with pytest.raises(ValueError, match="CUDA"):
        moe.expert_linear(x, wq[None], ws[None], torch.zeros(2, dtype=torch.int32))
    for tensor in (x.float().requires_grad_(), ):
        with pytest.raises(RuntimeError, match="no gradient"):
            linear.linear_w8a8(tensor, wq, ws)
        with pytest.raises(RuntimeError, match="no gradient"):
            moe.expert_linear(tensor, wq[None], ws[None], None)
    with pytest.raises(RuntimeError, match="no gradient"):
        linear.linear_w8a8(x, wq, ws, torch.zeros(16, requires_grad=True))


def test_frozen_linear_cast_leaves_the_scales():
    from triton_int8_b200.linear import Int8FrozenLinear
    scale = torch.rand(16)
    frozen = Int8FrozenLinear(torch.zeros(16, 32, dtype=torch.int8), scale.clone(), torch.zeros(16)).to(torch.bfloat16)
    assert torch.equal(frozen.weight_scale, scale) and frozen.bias.dtype == torch.bfloat16 and frozen.weight_q.dtype == torch.int8
    assert torch.equal(frozen.state_dict()["weight_scale"], scale)
