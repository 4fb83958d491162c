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
