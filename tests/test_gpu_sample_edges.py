"""The sampler at the ends of its ranges: temperatures up to the largest number."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from test_gpu_sample import check, run, settings

pytestmark = pytest.mark.gpu

LARGEST = float(np.finfo(np.float32).max)


@pytest.fixture(scope="module")
def sampling(mlk):
    return importlib.import_module(mlk.__name__ + ".sampling")


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [300, 5000, 128256])
@pytest.mark.parametrize("t", [1e37, 2e37, 1e38, LARGEST])
def test_a_masked_logit_is_not_chosen_at_the_highest_temperatures(mlk, sampling, t, V, act):
    """Ten logits are left, which weigh the same; cuts that reach past them, few rows and many."""
    rng = np.random.default_rng(V)
    for rows in (12, 290):
        x = np.full((rows, V), -np.inf, np.float32)
        for r in range(rows):
            x[r, rng.choice(V, 10, replace=False)] = rng.standard_normal(10) * 3
        u = np.resize(np.float32([0.05, 0.55, 0.95, 1 - 2.0 ** -24]), rows)
        how = settings(rows, t=t, u=u, k=list(np.resize([40, 0, 40, 7, 20000, 40], rows)),
                       p=list(np.resize([1, 1, 1, 1, 0.93, 0.93, 0.55], rows)),
                       m=list(np.resize([0, 0.1, 0.2, 0, 0], rows)))
        check(x, how, run(mlk, sampling, x, how, act), act, 1.0)
