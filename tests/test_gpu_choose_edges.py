"""DeviceModel.choose with settings that float32 and int32 do not hold as they are."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from conftest import tiny_model
from test_gpu_sample import define

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fwd(mlk):
    return importlib.import_module(mlk.__name__ + ".forward")


def test_uniform_numbers_next_to_one(fwd):
    """float64 numbers below 1 whose nearest float32 is 1: the largest float32 below 1."""
    model, tokens, _, _ = tiny_model()
    dm = fwd.DeviceModel(model)
    below = float(np.nextafter(np.float32(1), np.float32(0)))
    for u in (1 - 2.0 ** -53, 1 - 2.0 ** -26):
        want = define(dm.forward(tokens).astype(np.float64), 1.0, 0, 1.0, 0.0, below)
        got = dm.choose(tokens, u)
        assert got[0] == dm.choose(tokens, below)[0]
        if want[2]:
            assert got[0] == want[0]
    ids, _ = dm.choose(tokens, np.array([0.25, 1 - 2.0 ** -40]))
    assert ids[1] == dm.choose(tokens, [0.25, below])[0][1]
    for u in (1.0, 1 + 2.0 ** -30, -2.0 ** -60, float("nan")):
        with pytest.raises(ValueError, match="no token to choose"):
            dm.choose(tokens, u)


def test_top_k_past_32_bits(fwd):
    """A top-k of more tokens than int32 counts keeps all; a negative one does too."""
    model, tokens, _, _ = tiny_model()
    dm = fwd.DeviceModel(model)
    want = dm.choose(tokens, [0.9, 0.95])
    for k in (2 ** 40, 2 ** 32 + 1, -2 ** 40, np.array([2 ** 32 + 1, 2 ** 63 - 1]), [2 ** 32 + 1, -2 ** 62]):
        got = dm.choose(tokens, [0.9, 0.95], top_k=k)
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a, b)
