"""CPU: AdamW around the engine -- the step count of a checkpoint."""

import numpy as np
import pytest

from wide_deep_amd.plan import steps_of_powers


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.9, 0.99), (0.9, 0.9999), (0.9, 0.99999), (0.99, 0.5), (0.9, 0.0), (0.0, 0.9)])
def test_steps_from_the_powers_of_a_checkpoint(betas):
    """The running fp32 products of every step are told apart, far behind where their logarithms are a step off."""
    top = max(betas)
    products = np.multiply.accumulate(np.full(400000, top, dtype=np.float32))
    n = int((products >= 2.0 ** -126).sum())
    low = np.multiply.accumulate(np.full(400000, min(betas), dtype=np.float32))
    for t in [0, 1, 2, 207, 208, 3043, 3044, 5000, 65535, 65536, 70000, 131072, 399999]:
        powers = [float(products[t] if b == top else low[t]) for b in betas]
        got = steps_of_powers(betas, powers)
        if t < n:
            assert got == t
        else:
            assert top ** got < 2.0 ** -100
    assert steps_of_powers(betas, list(betas)) == 0 and steps_of_powers((0.0, 0.0), (0.0, 0.0)) == 0
