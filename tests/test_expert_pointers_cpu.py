"""Pointers that the entry points of the expert layers refuse, whatever else is asked for: a kernel would read through them.  No device
is needed: what passes the checks ends in an architecture or CUDA error."""
import ctypes

import pytest
import torch

NO_DEVICE = (-3, -4)
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="pointers of no device: checks what is refused before a launch")


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


def _combine_backward(lib, p, **change):
    a = dict(rows=0, weights=0, pos=0, src=0, dy=0, n_rows=8, tokens=4, cols=8, k=2, dtype=0, wdtype=0, drows=0, dweights=0)
    a.update(change)
    at = lambda off: None if off is None else p + off  # noqa: E731
    return lib.i8l_combine_backward(at(a["rows"]), at(a["weights"]), at(a["pos"]), at(a["src"]), at(a["dy"]), a["n_rows"], a["tokens"], a["cols"],
                                    a["k"], a["dtype"], a["wdtype"], at(a["drows"]), at(a["dweights"]), None)


@pytest.mark.parametrize("cols", [8, 7])   # rows of whole 16 bytes and odd ones
@pytest.mark.parametrize("only", [{}, dict(drows=None), dict(dweights=None)])
def test_gradients_of_combine_need_src(lib, p, cols, only):
    assert _combine_backward(lib, p, cols=cols, **only) in NO_DEVICE
    assert _combine_backward(lib, p, cols=cols, src=None, **only) == -6


def test_without_rows_there_is_no_src(lib, p):
    assert _combine_backward(lib, p, n_rows=0, src=None, rows=None, drows=None) in NO_DEVICE


@pytest.mark.parametrize("name", ["rows", "weights", "pos", "src", "dy", "drows", "dweights"])
def test_gradients_of_combine_want_aligned_pointers(lib, p, name):
    assert _combine_backward(lib, p, **{name: 2}, dtype=2, wdtype=2) == -2


@pytest.mark.parametrize("name", ["x", "ids", "out", "offsets", "pos", "src", "ws"])
@pytest.mark.parametrize("tokens", [4, 1000])   # one launch, three
def test_sort_wants_aligned_pointers(lib, p, name, tokens):
    a = dict(x=0, ids=0, out=0, offsets=0, pos=0, src=0, ws=0)

    def run(a):
        return lib.i8l_sort_tokens(p + a["x"], p + a["ids"], 0, tokens, 8, 2, 4, 1, 2, 2000, p + a["out"], p + a["offsets"], p + a["pos"],
                                   p + a["src"], p + a["ws"], 4096, None)
    assert run(a) in NO_DEVICE
    assert run(dict(a, **{name: 2})) == -2


@pytest.mark.parametrize("name", ["x", "wq", "ws", "offsets", "bias", "y", "work", "status"])
@pytest.mark.parametrize("rows", [2, 40])
def test_the_product_for_serving_wants_aligned_pointers(lib, p, name, rows):
    a = dict(x=0, wq=0, ws=0, offsets=0, bias=0, y=0, work=0, status=0)

    def run(a):
        return lib.i8l_token_linear(p + a["x"], p + a["wq"], p + a["ws"], p + a["offsets"], p + a["bias"], p + a["y"], rows, 4, 16, 32, 0,
                                    p + a["work"], 1 << 14, p + a["status"], None)
    assert run(a) in NO_DEVICE
    assert run(dict(a, **{name: 2})) == -2
