"""GPU: calls of the operators around a step's matrix products at the borders of what
include/meshgpt.h allows, against plain 64-bit forms (tests/steps_lib.py)."""
import math

import numpy as np
import pytest

import grokking_abmod_amd as G
import operators_lib as L
from test_gpu_steps import KINDS, sampled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [1, 5, 200, 700, 9000, 40003, 90003])
@pytest.mark.parametrize("kind", KINDS)
def test_greedy_rows_look_at_no_filter_and_no_number(kind, vocab):
    """At temperature 0 settings that are no numbers do not matter, nor do their values."""
    rng = np.random.default_rng(vocab)
    choices = [0.0, 0.5, 7.0, -1.0, math.nan, math.inf]
    p, m = (a.ravel() for a in np.meshgrid(choices, choices))
    rows = len(p)
    z = L.stored(rng.normal(size=(rows, vocab)), kind)
    with L.Device() as dev:
        for kw in (dict(top_p=p, min_p=m), dict(top_p=p), dict(min_p=m), dict(top_p=p, min_p=m, top_k=np.full(rows, 3))):
            tokens, logprob, _ = sampled(dev, z, kind, temperature=np.zeros(rows), u=rng.choice([math.nan, 2.0, 0.5], rows), **kw)
            assert np.array_equal(tokens, np.argmax(L.values(z, kind), 1))
            assert not logprob.any()
