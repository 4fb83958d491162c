"""Numbers of experts and alignments above what the sort takes, from Python: refused before anything of that size is made."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("change", [dict(experts=1025), dict(experts=20000), dict(experts=70000), dict(experts=2 ** 32 + 5), dict(align=65537),
                                    dict(align=2 ** 40), dict(experts=2 ** 62)])
def test_too_many(change):
    from triton_int8_b200 import I8LError, moe
    x, ids = torch.zeros(1025, 8, device=DEV), torch.zeros(1025, 2, dtype=torch.int64, device=DEV)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    with pytest.raises(I8LError, match="SHAPE"):
        moe.sort_tokens(x, ids, **dict(dict(experts=4, align=1), **change))
    assert torch.cuda.max_memory_allocated() == before
