"""CPU: AdamW around the engine -- the step count of a checkpoint, and what is told of skipped steps."""

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


def test_skipped_steps_are_told(capsys):
    """What a training run skipped is told once, what a checkpoint brought along is not."""
    from types import SimpleNamespace
    from wide_deep_amd.estimator import WideAndDeepClassifier
    opt = SimpleNamespace(max_norm=1.0, skipped=2)
    est = WideAndDeepClassifier(None, engine=SimpleNamespace(adamw=opt))

    def told():
        est._tell_skipped()
        return capsys.readouterr().out

    assert told() == ""
    opt.skipped = 5
    assert told().startswith("WARNING: 3 train steps") and told() == ""
    opt.skipped = 6
    assert told().startswith("WARNING: 1 train steps")
    opt.max_norm, opt.skipped = None, 9
    assert told() == ""
    for engine in (SimpleNamespace(adamw=None), SimpleNamespace()):
        est = WideAndDeepClassifier(None, engine=engine)
        assert told() == ""
