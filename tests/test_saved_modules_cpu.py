"""Modules with experts can be pickled, saved whole and copied, and what is loaded into a copy drops its frozen weights."""
import copy
import io
import pickle

import pytest
import torch

from triton_int8_b200 import moe
from triton_int8_b200.decoder_layer import DecoderLayer


def _saved(m):
    buf = io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


@pytest.mark.parametrize("again", [lambda m: pickle.loads(pickle.dumps(m)), _saved, copy.deepcopy])
@pytest.mark.parametrize("make", [lambda: moe.Int8MoE(128, 128, experts=2, top_k=1), lambda: DecoderLayer(hidden=128, heads=2, mlp=128, experts=2)])
def test_copies(again, make):
    torch.manual_seed(0)
    first, other = make(), make()
    second = again(first)
    assert set(second.state_dict()) == set(first.state_dict())
    assert all(torch.equal(v, second.state_dict()[k]) for k, v in first.state_dict().items())
    layer = second if isinstance(second, moe.Int8MoE) else second.moe
    layer._frozen = ()
    second.load_state_dict(other.state_dict())
    assert layer._frozen is None
