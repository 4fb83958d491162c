"""More experts than the sort takes: an error, whatever their number.  No device is needed."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _child(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=240)


@pytest.mark.parametrize("experts", [1025, 16384, 16385, 65536, 2 ** 31 - 1, -1])
@pytest.mark.parametrize("tokens", [1, 1025, 1 << 30, 1 << 62])
def test_workspace_of_what_is_refused(experts, tokens):
    """A chunk of choices was doubled until the counts of all chunks fit, which none does with more than 16384 experts."""
    r = _child(f"from triton_int8_b200 import _lib; print(_lib.load().i8l_sort_workspace({tokens}, 2, {experts}))")
    assert r.returncode == 0 and r.stdout.strip() == "0", (r.returncode, r.stdout, r.stderr[-500:])


def test_workspace_of_what_is_taken():
    from triton_int8_b200 import _lib
    lib = _lib.load()
    assert lib.i8l_sort_workspace(1 << 29, 2, 1024) == 16 * 1024 * 4 and lib.i8l_sort_workspace(1025, 64, 1) == 257 * 4
    assert lib.i8l_sort_workspace((1 << 29) + 1, 2, 1024) == 0 and lib.i8l_sort_workspace(1025, 65, 1) == 0
