"""GPU: an engine with dnn_optimizer AdamW goes on from a checkpoint as the one that wrote it -- late steps, skipped steps, files without a count."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _engine(seed, betas=(0.9, 0.99), max_norm=0.5, model_type="wide_deep"):
    from wide_deep_amd.engine import WideDeepEngine
    from wide_deep_amd.plan import criteo_spec
    s = criteo_spec(n_dense=3, n_sparse=5, buckets=40, dim=16, hidden=(32, 16), model_type=model_type)
    s.dnn_opt = ("AdamW", 0.01) + betas + (1e-8, 0.1, max_norm)
    return WideDeepEngine(s, max_batch=64, seed=seed)


def _batch(eng, seed):
    from wide_deep_amd import synth
    return synth.to_device_ids(eng.plan, synth.make_raw_batch(eng.plan, 64, seed=seed, pos_rate=0.4))


def _powers(betas, steps):
    """beta^(steps + 1) of both as the running fp32 products that the tables' Adam keeps."""
    return [float(np.multiply.accumulate(np.full(steps + 1, b, dtype=np.float32))[-1]) for b in betas]


def _go_on_alike(a, b):
    for k in range(2):
        a.train_step(_batch(a, 50 + k))
        b.train_step(_batch(b, 50 + k))
        torch.cuda.synchronize()
        for x, y in ((a.P, b.P), (a.adamw.m, b.adamw.m), (a.adamw.v, b.adamw.v), (a.emb, b.emb)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("betas,steps", [((0.9, 0.9999), 5000), ((0.9, 0.99999), 1000), ((0.9, 0.999), 200000), ((0.99, 0.5), 300), ((0.9, 0.0), 7)])
def test_late_steps_resume(betas, steps):
    a, c = _engine(4, betas), _engine(77, betas)
    a.train_step(_batch(a, 1))
    a.adamw.set_step(steps)
    a.pow["dnn"].copy_(torch.tensor(_powers(betas, steps)))
    state = a.export_state()
    assert a.state_shapes() == {k: tuple(v.shape) for k, v in state.items()}
    c.import_state(state)
    assert c.adamw.step_count == a.adamw.step_count == steps
    _go_on_alike(a, c)
    # a file without the count: from the running products, as long as one of them has not left fp32
    del state["dnn/AdamW/steps"]
    d = _engine(78, betas)
    d.import_state(state)
    if max(_powers(betas, steps)) > 2.0 ** -126:
        assert d.adamw.step_count == steps
    else:                                        # both corrections are 1 to the last bit
        assert max(b ** d.adamw.step_count for b in betas) < 2.0 ** -25


def test_skipped_steps_are_in_the_checkpoint():
    """A step whose norm is not finite leaves the dense parameters and their step count alone; the tables' Adam goes on.  An engine that
    restores such a state goes on as the saved one."""
    from wide_deep_amd import capi
    a, c = _engine(4), _engine(77)
    a.train_step(_batch(a, 1))
    for _ in range(3):
        was = a.P.clone()
        a.G.fill_(math.inf)
        a.adamw.step(lr=0.01)
        capi.call("wd_adam_tick", capi.ptr(a.pow["dnn"]), 0.9, 0.99, None)
        torch.cuda.synchronize()
        assert torch.equal(a.P, was)
    a.train_step(_batch(a, 2))
    assert (a.adamw.step_count, a.adamw.skipped) == (2, 3)
    c.import_state(a.export_state())
    assert (c.adamw.step_count, c.adamw.skipped) == (2, 3)
    _go_on_alike(a, c)


def test_a_state_without_counters_leaves_the_count_alone():
    a = _engine(4)
    for k in range(3):
        a.train_step(_batch(a, k))
    a.adamw.set_step(10)
    state = {k: v for k, v in a.export_state().items() if k not in ("dnn/AdamW/steps", "beta1_power", "beta2_power", "global_step")}
    a.import_state(state)
    assert a.adamw.step_count == 10


def test_max_norm_guards_the_dense_parameters_alone():
    """Inputs of 1e30: the kernels' gradients have no finite norm, the tables' gradients are ordinary.  The towers stay, the tables step."""
    a = _engine(4)
    a.train_step(_batch(a, 1))
    bt = _batch(a, 2)
    bt.dense[:, 1] = 1e30                        # every example: one at least is answered wrongly through a unit that is on
    P, emb = a.P.clone(), a.emb.clone()
    a.train_step(bt)
    torch.cuda.synchronize()
    assert a.adamw.skipped == 1 and a.adamw.step_count == 1 and not math.isfinite(float(a.adamw.grad_norm))
    assert torch.equal(a.P, P) and not torch.equal(a.emb, emb) and bool(a.emb.isfinite().all())
