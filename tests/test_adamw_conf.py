"""CPU: AdamW around the engine -- `dnn_optimizer: AdamW` in model.yaml (by name, as a constructor, its rate's decay, what is refused) and the
step count of a checkpoint."""
import math
import shutil

import numpy as np
import pytest
import yaml

from wide_deep_amd import build_estimator as BE
from wide_deep_amd.build_estimator import opt_tuple, parse_optimizer
from wide_deep_amd.plan import steps_of_powers
from wide_deep_amd.read_conf import Config, conf_dir


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


def test_the_rate_of_an_adamw_given_by_name_decays(tmp_path):
    """lr_decay applies to optimizers given by name: AdamW as any other; a constructor keeps its own rate."""
    base = tmp_path / "conf"
    shutil.copytree(conf_dir(), base)
    tr = yaml.safe_load(open(base / "train.yaml"))
    tr["train"]["lr_decay"] = True
    yaml.safe_dump(tr, open(base / "train.yaml", "w"))
    m = yaml.safe_load(open(base / "model.yaml"))
    got = {}
    for name in ("Adam", "AdamW", " AdamW ", "AdamW(0.002)"):
        m["dnn_optimizer"] = name
        yaml.safe_dump(m, open(base / "model.yaml", "w"))
        conf = Config(base_dir=str(base))
        spec = BE.build_model_spec(conf, "wide_deep")
        got[name] = spec.lr_decay
        assert spec.dnn_opt[0] == name.strip().split("(")[0]
    steps = conf.train["num_examples"] / conf.train["batch_size"]
    assert got["Adam"] == got["AdamW"] == got[" AdamW "] == {"dnn": (0.8, steps)} and got["AdamW(0.002)"] is None


@pytest.mark.parametrize("text,message", [
    ("AdamW(lr=0.0003)", "lr"), ("AdamW(0.001, betas=(0.9, 0.95))", "betas"), ("AdamW(0.001, eps=1e-6)", "eps"), ("AdamW(0.001, state_bits=8)", "state_bits"),
    ("AdamW(0.001, 0.9, 0.95)", "by name"), ("AdamW(0.001, learning_rate=0.002)", "learning_rate"), ("AdamW(**{'beta1': 0.8})", "by name"),
    ("AdamW(0.001, max_norm=0)", "max_norm"), ("AdamW(0.001, max_norm=-1.0)", "max_norm"), ("AdamW(0.001, weight_decay=-1)", "weight_decay"),
    ("AdamW(0.001, beta1=1.0)", "beta1"), ("AdamW(0.001, beta2=-0.1)", "beta2"), ("AdamW(0.001, epsilon=-1e-8)", "epsilon")])
def test_arguments_that_would_be_dropped_or_cannot_be_are_refused(text, message):
    with pytest.raises(ValueError, match=message):
        opt_tuple(*parse_optimizer(text, 0.05))


def test_arguments_that_are_taken():
    assert opt_tuple(*parse_optimizer("AdamW()", 0.05)) == ("AdamW", 0.001, 0.9, 0.999, 1e-8, 0.01, None)
    assert opt_tuple(*parse_optimizer("optim.AdamW(learning_rate=0.01, beta1=0.8, beta2=0.9, epsilon=1e-6, weight_decay=0, max_norm=None)", 0.05)) == (
        "AdamW", 0.01, 0.8, 0.9, 1e-6, 0.0, None)
    assert opt_tuple(*parse_optimizer("AdamW(0.01, max_norm=1e999)", 0.05))[6] == math.inf
    # the reference's constructors stay as they were
    assert opt_tuple(*parse_optimizer("tf.train.AdamOptimizer(0.01, name='x')", 0.05)) == ("Adam", 0.01, 0.9, 0.999, 1e-8)
