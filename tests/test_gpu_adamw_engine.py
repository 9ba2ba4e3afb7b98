"""GPU: dnn_optimizer AdamW -- the engine's dense parameters through wd_adamw_step (decay on kernels, clipping by their norm), its embedding
tables through Adam -- against the formula in 64 bits from the state before each step; u = 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
OPT = ("AdamW", 0.01, 0.9, 0.99, 1e-8, 0.1, 0.5)
SHAPES = {"chain": dict(n_dense=16, n_sparse=3, buckets=300, dim=16, hidden=(64, 32)), "layers": dict(n_dense=3, n_sparse=5, buckets=40, dim=16, hidden=(32, 16), mode="resnet")}


def _spec(shape="layers", opt=OPT, **kw):
    from wide_deep_amd.plan import criteo_spec
    s = criteo_spec(**{**SHAPES[shape], **kw})
    s.dnn_opt = opt
    return s


def _batch(eng, seed, B=64):
    from wide_deep_amd import synth
    return synth.to_device_ids(eng.plan, synth.make_raw_batch(eng.plan, B, seed=seed, pos_rate=0.4))


@pytest.mark.parametrize("shape,max_norm", [("chain", 0.5), ("layers", 0.5), ("layers", None), ("chain", 1e6)])
def test_train_steps(shape, max_norm):
    """Kernels decay, vectors do not; the tables move as with Adam: the same bits after the first step, whose gradients are the same."""
    from wide_deep_amd.engine import WideDeepEngine
    opt = OPT[:6] + (max_norm,)
    eng, adam = WideDeepEngine(_spec(shape, opt), max_batch=64, seed=2), WideDeepEngine(_spec(shape, ("Adam",) + OPT[1:5]), max_batch=64, seed=2)
    assert bool(eng.chain) == (shape == "chain") and eng.adamw.state_bits == 32
    lr, b1, b2, eps, decay = OPT[1:6]
    for t in (1, 2, 3):
        before = {k: v.clone() for k, v in dict(P=eng.P, m=eng.adamw.m, v=eng.adamw.v).items()}
        eng.train_step(_batch(eng, t))
        if t == 1:
            adam.train_step(_batch(adam, t))
            torch.cuda.synchronize()
            assert torch.equal(eng.emb, adam.emb) and torch.equal(eng.emb_a, adam.emb_a) and torch.equal(eng.wide, adam.wide)
        grads = eng._dense_tensors(eng.G)
        norm = math.sqrt(sum(float(g.double().square().sum()) for g, _ in grads))
        coef = max_norm / max(norm, max_norm) if max_norm else 1.0
        assert not max_norm or abs(float(eng.adamw.grad_norm) - norm) <= 10 * U * norm
        for (p0, kernel), (p1, _), (g, _), a in zip(eng._dense_tensors(before["P"]), eng._dense_tensors(eng.P), grads, eng.adamw.starts):
            part = slice(a, a + g.numel())
            m0, v0, g = before["m"][part].double(), before["v"][part].double(), g.double() * coef
            m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
            tm = 6 * U * (b1 * m0.abs() + (1 - b1) * g.abs())
            root = torch.sqrt(v / (1 - b2 ** t)) + eps
            d = decay * p0.double() if kernel else 0.0 * p0.double()
            want = p0.double() - lr * (m / (1 - b1 ** t) / root + d)
            # as the operator's own tests: 16 u of the update's terms, u of the parameter
            tol = 16 * U * lr * ((m.abs() + tm / U / 16) / (1 - b1 ** t) / root + d.abs()) + U * p0.double().abs() + 1e-45
            assert bool(((p1.double() - want).abs() <= tol).all()), (t, kernel, float(((p1.double() - want).abs() / tol).max()))
    assert eng.adamw.step_count == 3


@pytest.mark.parametrize("shape", ["chain", "layers"])
def test_captured_steps_and_checkpoints(shape):
    """A captured step replays the eager ones bit for bit; an engine that takes over the other's state goes on as it does."""
    from wide_deep_amd.engine import WideDeepEngine
    a, b = WideDeepEngine(_spec(shape), max_batch=64, seed=4), WideDeepEngine(_spec(shape), max_batch=64, seed=4)
    bta, btb = _batch(a, 9), _batch(b, 9)
    replay = a.capture_train_step(bta, warmup=1)
    b.train_step(btb)
    for _ in range(3):
        replay()
        b.train_step(btb)
        torch.cuda.synchronize()
        assert torch.equal(a.P, b.P) and torch.equal(a.adamw.m, b.adamw.m)
    state = b.export_state()
    assert b.state_shapes() == {k: tuple(v.shape) for k, v in state.items()}
    key = "dnn/dnn_1/hiddenlayer_0/kernel"
    assert float(state[key + "/Adam"].abs().sum()) > 0 and float(state[key + "/Adam_1"].abs().sum()) > 0
    c = WideDeepEngine(_spec(shape), max_batch=64, seed=77)
    c.train_step(_batch(c, 3))
    c.import_state(state)
    assert c.adamw.step_count == b.adamw.step_count == 4
    for k in range(2):
        b.train_step(btb)
        c.train_step(btb)
        torch.cuda.synchronize()
        for x, y in ((b.P, c.P), (b.adamw.m, c.adamw.m), (b.adamw.v, c.adamw.v), (b.emb, c.emb)):
            assert torch.equal(x, y)


def test_learning_rates_conf_and_refusals():
    from wide_deep_amd.build_estimator import opt_tuple, parse_optimizer
    from wide_deep_amd.engine import WideDeepEngine
    assert opt_tuple(*parse_optimizer("AdamW", 0.05)) == ("AdamW", 0.05, 0.9, 0.999, 1e-8, 0.01, None)
    text = "AdamW(0.002, beta2=0.95, weight_decay=0.1, max_norm=1)"
    assert opt_tuple(*parse_optimizer(text, 0.05)) == ("AdamW", 0.002, 0.9, 0.95, 1e-8, 0.1, 1.0)
    s = _spec()
    s.lin_opt = OPT
    with pytest.raises(ValueError, match="optimizer of the dnn scope"):
        WideDeepEngine(s, max_batch=64)
    for opt in (OPT, OPT[:6] + (None,)):
        s = _spec(opt=opt)
        s.activation = "crelu"
        if opt[6]:
            with pytest.raises(ValueError, match="tied halves"):       # the norm would count a kernel twice
                WideDeepEngine(s, max_batch=64)
        else:
            eng = WideDeepEngine(s, max_batch=64, seed=1)
            eng.train_step(_batch(eng, 1))
            assert eng.adamw.step_count == 1 and bool(eng.P.isfinite().all())
    eng = WideDeepEngine(_spec(), max_batch=64, seed=1)
    eng.set_learning_rates(dnn=0.0)
    p = eng.P.clone()
    eng.train_step(_batch(eng, 1))
    assert torch.equal(eng.P, p) and eng.adamw.step_count == 1
    eng = WideDeepEngine(_spec(model_type="wide"), max_batch=64, seed=1)       # no dnn scope
    eng.train_step(_batch(eng, 1))
    assert eng.adamw is None and "beta1_power" not in eng.export_state()


def _worker(rank, world, port, kind, q):
    import tests.test_gpu_dist as T
    spec = T._spec(kind)
    spec[0].dnn_opt = OPT
    T._spec = lambda k: spec
    T._worker(rank, world, port, kind, q)


def test_two_ranks_take_the_steps_of_one():
    from tests.test_gpu_dist import _run
    _run(_worker, "adam")
