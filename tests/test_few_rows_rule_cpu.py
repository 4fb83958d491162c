"""Which sizes of the product for serving the kernels for few rows take: they need no workspace, the tensor cores do."""
import pytest


@pytest.mark.parametrize("few,rows,experts,N,K", [
    (True, 5, 1, 4096, 4096), (True, 5, 1, 4104, 4096), (True, 8, 1, 6144, 4096), (False, 8, 1, 6152, 4096),     # weights
    (True, 4, 1, 10240, 4096), (False, 4, 1, 10248, 4096), (True, 4, 4, 8192, 2048), (True, 2, 8, 11008, 4096),
    (True, 1, 1, 8, 32768), (False, 1, 1, 8, 32784), (False, 2, 1, 8, 16400), (False, 3, 1, 8, 8208), (False, 5, 1, 8, 4112), (False, 8, 1, 8, 4112),   # K
    (True, 8, 8, 192, 1024), (False, 8, 8, 200, 1024), (True, 8, 1, 11008, 2048), (False, 6, 64, 1408, 2048),    # experts
    (False, 9, 1, 8, 16)])
def test_rule(few, rows, experts, N, K):
    from triton_int8_b200 import _lib
    assert (_lib.load().i8l_token_linear_workspace(rows, experts, N, K) == 0) == few
