"""DeviceModel.choose: the sampler behind a forward pass, against the definition on the
logits that forward() returns for the same tokens."""
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


def f32(x):
    return float(np.float32(x))


def test_choose_is_the_definition_on_the_forward_logits(mlk, fwd):
    model, tokens, _, _ = tiny_model()
    dm = fwd.DeviceModel(model)
    logits = dm.forward(tokens, all_logits=True).astype(np.float64)
    rng = np.random.default_rng(1)
    n = len(tokens)
    for how in (dict(), dict(temperature=0.0), dict(temperature=0.7, top_p=0.9), dict(top_k=5),
                dict(temperature=1.3, top_k=40, top_p=0.95, min_p=0.02)):
        u = rng.random(n).astype(np.float32)
        ids, shares = dm.choose(tokens, u, **how)
        for t in range(n):
            token, prob, sure = define(logits[t], f32(how.get("temperature", 1.0)), how.get("top_k", 0),
                                       f32(how.get("top_p", 1.0)), f32(how.get("min_p", 0.0)), f32(u[t]))
            assert sure and ids[t] == token
            assert abs(shares[t] - prob) <= 2.0 ** -23 * prob
        # one row: the last token's logits alone, which other kernels may round otherwise
        one, share = dm.choose(tokens, u[-1], **how)
        token, prob, sure = define(dm.forward(tokens).astype(np.float64), f32(how.get("temperature", 1.0)),
                                   how.get("top_k", 0), f32(how.get("top_p", 1.0)),
                                   f32(how.get("min_p", 0.0)), f32(u[-1]))
        assert sure and one == token and isinstance(one, int)
        assert abs(share - prob) <= 2.0 ** -23 * prob
    # settings row by row, on a stream, after a prompt at later positions
    dm.forward(tokens[:4])
    stream = mlk.Stream()
    want = fwd.DeviceModel(model)
    want.forward(tokens[:4])
    logits = want.forward(tokens[4:7], pos0=4, all_logits=True).astype(np.float64)
    k, t, u = [3, -1, 0], [0.5, 0.0, 2.0], [0.9, 0.9, 0.1]
    ids, _ = dm.choose(tokens[4:7], u, temperature=t, top_k=k, pos0=4, stream=stream.handle)
    for i in range(3):
        assert ids[i] == define(logits[i], f32(t[i]), k[i], 1.0, 0.0, f32(u[i]))[0]


def test_choose_refusals(fwd):
    model, tokens, _, _ = tiny_model()
    dm = fwd.DeviceModel(model)
    with pytest.raises(ValueError, match="uniform numbers"):
        dm.choose(tokens[:2], [0.1, 0.2, 0.3])
    with pytest.raises(ValueError, match="uniform numbers"):
        dm.choose(tokens[:2], [])
    for kw in (dict(temperature=-1.0), dict(top_p=float("nan"))):
        with pytest.raises(ValueError, match="no token to choose"):
            dm.choose(tokens, 0.5, **kw)
    with pytest.raises(ValueError, match="no token to choose"):
        dm.choose(tokens, 1.0)
    assert dm.choose(tokens, 0.0)[0] == dm.forward(tokens).argmax()
