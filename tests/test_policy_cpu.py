"""CPU: the policy heads and AdamW refuse what they cannot do before anything touches a device (csrc/policy_loss.hip, csrc/adamw.hip,
wide_deep_amd/policy.py, optim.py), and the packed argument records are as long as the structs of include/wd_hip.h."""
import os
import re

import numpy as np
import pytest
import torch

from wide_deep_amd import capi, optim, policy

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SIZE = {"int64_t": 8, "uint64_t": 8, "double": 8, "float": 4, "int32_t": 4, "uint32_t": 4}


def _struct(name):
    """Fields of a struct of the header in order: (name, bytes)."""
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "wd_hip.h")).read(), flags=re.S)
    body = re.search(r"typedef struct \w+ \{([^}]*)\} %s;" % name, src).group(1)
    out = []
    for line in filter(None, (x.strip() for x in body.split(";"))):
        first, *more = line.split(",")
        kind, field = re.match(r"(?:const )?(\w+)\s+(\*?\w+)$", first.strip()).groups()
        for f in [field] + [m.strip() for m in more]:
            out.append((f.lstrip("*"), 8 if f.startswith("*") else SIZE[kind]))
    return out


@pytest.mark.parametrize("name,fmt", [("wd_seq_rows_t", policy._ROWS), ("wd_pref_t", policy._PREF), ("wd_policy_t", policy._POLICY),
                                      ("wd_adamw_t", optim._OPTS)])
def test_packed_records_match_the_header(name, fmt):
    widths = [8 if c in "Qqd" else 4 for c in fmt.format.lstrip("=")]
    assert widths == [b for _, b in _struct(name)]
    assert all(sum(widths[:i]) % w == 0 for i, w in enumerate(widths)) and fmt.size == sum(widths)       # no padding in between


def test_tensor_and_state_records_match_the_header():
    assert [(n, optim._TENSOR.fields[n][0].itemsize) for n in optim._TENSOR.names][:6] == _struct("wd_adamw_tensor_t")[:6]
    state = _struct("wd_adamw_state_t")
    at = {n: sum(b for _, b in state[:k]) // 4 for k, (n, _) in enumerate(state)}
    assert sum(b for _, b in state) == 48 and (at["step"], at["skipped"], at["norm"]) == (0, 2, 10)       # what optim.py reads
    src = open(os.path.join(ROOT, "include", "wd_hip.h")).read()
    for name, value in (("BLOCK", optim.BLOCK), ("CHUNK", optim.CHUNK), ("PARTIALS", optim.PARTIALS), ("TICKETS", optim.TICKETS)):
        assert int(re.search(r"#define WD_ADAMW_%s (\d+)" % name, src).group(1)) == value


def _rows(rows=8, vocab=16, seqs=2, dtype=0, ld=None, logits=1 << 20, targets=64, offs=64):
    return policy._ROWS.pack(logits, vocab if ld is None else ld, rows, vocab, targets, offs, seqs, dtype, 0)


@pytest.mark.parametrize("kw,message", [(dict(rows=-1), "bad sizes"), (dict(vocab=0, ld=4), "bad sizes"), (dict(seqs=-1), "bad sizes"),
                                        (dict(dtype=3), "bad element type"), (dict(ld=15), "row stride"), (dict(targets=0), "null pointer"),
                                        (dict(offs=0), "null pointer"), (dict(logits=0), "null pointer"), (dict(logits=2), "not aligned"),
                                        (dict(rows=1 << 31), "2\\^30"), (dict(vocab=1 << 31), "2\\^30")])
def test_rows_are_checked(kw, message):
    with pytest.raises(capi.WdError, match="wd_seq_logp failed .*" + message):
        capi.call("wd_seq_logp", _rows(**kw), 0, 64, 64, 64, None)
    assert capi.call("wd_policy_workspace_floats", _rows(**kw)) < 0


def _pref(loss=64, pair=64, diff=64, seq=64, tok=64, grad=0, ld=16, beta=0.1, margin=0.0, smooth=0.0, kind=0):
    return policy._PREF.pack(0, 0, loss, pair, diff, seq, tok, grad, ld, beta, margin, smooth, 1.0, 1.0, kind, 0, 0)


@pytest.mark.parametrize("rows,kw,message", [(dict(seqs=3), {}, "odd number"), ({}, dict(kind=2), "bad loss kind"), ({}, dict(beta=0.0), "beta"),
                                             ({}, dict(beta=float("nan")), "beta"), ({}, dict(smooth=0.5), "label_smoothing"),
                                             ({}, dict(smooth=float("nan")), "label_smoothing"), ({}, dict(kind=1, margin=0.1), "logistic"),
                                             ({}, dict(loss=0), "null output"), ({}, dict(tok=0), "null output"), ({}, dict(diff=0), "null output"),
                                             ({}, dict(grad=64, ld=15), "row stride of the gradient"), ({}, dict(grad=66), "gradient not aligned")])
def test_preference_options_are_checked(rows, kw, message):
    with pytest.raises(capi.WdError, match="wd_pref_loss_fwd_bwd failed .*" + message):
        capi.call("wd_pref_loss_fwd_bwd", _rows(**rows), _pref(**kw), 64, None)


def _policy(old=64, ref=0, adv=64, sums=64, tok=64, grad=0, ld=16, low=0.2, high=0.2, kl=0.0, by_row=0, reduction=0):
    return policy._POLICY.pack(old, ref, adv, sums, tok, grad, ld, low, high, kl, 1.0, by_row, reduction, 0, 0)


@pytest.mark.parametrize("kw,message", [(dict(reduction=3), "bad reduction"), (dict(low=1.5), "clip range"), (dict(low=-0.1), "clip range"),
                                        (dict(high=float("nan")), "clip range"), (dict(kl=0.1), "reference policy"), (dict(old=0), "null pointer"),
                                        (dict(adv=0), "null pointer"), (dict(sums=0), "null pointer"), (dict(grad=64, ld=8), "row stride of the gradient")])
def test_policy_options_are_checked(kw, message):
    with pytest.raises(capi.WdError, match="wd_policy_loss_fwd_bwd failed .*" + message):
        capi.call("wd_policy_loss_fwd_bwd", _rows(), _policy(**kw), 64, None)


def _adamw(tensors=64, chunks=64, n=1, m=64, v=64, ms=64, rs=64, state=64, tickets=64, partials=64, b1=0.9, b2=0.999, eps=1e-8, norm=0.0, bits=32, gt=0, ct=2):
    return optim._OPTS.pack(tensors, chunks, n, m, v, ms, rs, state, tickets, partials, 0, b1, b2, 1e-3, eps, norm, 0, bits, gt, ct, 0)


@pytest.mark.parametrize("kw,message", [(dict(tensors=0), "null pointer"), (dict(n=0), "no chunks"), (dict(state=0), "null pointer"), (dict(tickets=0), "null pointer"), (dict(bits=16), "32 or in 8"),
                                        (dict(bits=8, ms=0), "scales"), (dict(gt=3), "gradient type"), (dict(ct=0), "copy"), (dict(b1=1.0), "betas"), (dict(m=72), "aligned to 16"), (dict(v=68, bits=8), "aligned to 16"),
                                        (dict(b2=float("nan")), "betas"), (dict(eps=-1.0), "betas"), (dict(norm=1.0, partials=0), "partials")])
def test_adamw_options_are_checked(kw, message):
    with pytest.raises(capi.WdError, match="wd_adamw_step failed .*" + message):
        capi.call("wd_adamw_step", _adamw(**kw), None)


def test_adamw_helpers_are_checked():
    for args in ((None, 64, 0, 0.9, 0.999), (64, None, 0, 0.9, 0.999), (64, 64, -1, 0.9, 0.999), (64, 64, 0, 1.0, 0.999)):
        with pytest.raises(capi.WdError, match="wd_adamw_set_step failed"):
            capi.call("wd_adamw_set_step", *args, None)
    with pytest.raises(capi.WdError, match="multiple of the block"):
        capi.call("wd_adamw_unpack", 64, 64, 64, 64, 65, 64, 64, 2, None)
    with pytest.raises(capi.WdError, match="bf16 or fp32"):
        capi.call("wd_adamw_unpack", 64, 64, 64, 64, 64, 64, 64, 1, None)
    with pytest.raises(capi.WdError, match="multiple of the block"):
        capi.call("wd_adamw_pack", 64, 64, 0, 64, 64, 64, 64, None)
    with pytest.raises(capi.WdError, match="aligned to 16"):
        capi.call("wd_adamw_unpack", 64, 64, 64, 64, 64, 64, 72, 0, None)
    with pytest.raises(capi.WdError, match="aligned to 16"):
        capi.call("wd_adamw_pack", 68, 64, 64, 64, 64, 64, 64, None)


def test_python_entry_points_refuse_before_the_device():
    z, t, o = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32), torch.tensor([0, 2, 4], dtype=torch.int32)
    for call in (lambda z: policy.sequence_logp(z, t, o), lambda z: policy.preference_loss(z, t, o), lambda z: policy.policy_loss(z, t, o, torch.zeros(4), torch.zeros(2))):
        with pytest.raises(capi.WdError, match="no CPU fallback"):
            call(z)
        for bad in (torch.zeros(4, 8, dtype=torch.float64), torch.zeros(8), torch.zeros(4, 0), torch.zeros(4, 16)[:, ::2], torch.zeros(1, 8).expand(4, 8), None):
            with pytest.raises(ValueError, match="logits"):
                call(bad)
    p = [torch.zeros(3, 5), torch.zeros(7)]
    g = [torch.zeros(3, 5), torch.zeros(7)]
    with pytest.raises(capi.WdError, match="no CPU fallback"):
        optim.AdamW(p, g)
    for kw, message in ((dict(params=[]), "at least one"), (dict(grads=g[:1]), "as many"), (dict(grads=[g[0], torch.zeros(8)]), "gradient 1"),
                        (dict(grads=[g[0], g[1].half()]), "gradient 1"), (dict(params=[p[0].double(), p[1]]), "parameter 0"),
                        (dict(params=[p[0].t().contiguous().t(), p[1]]), "parameter 0"), (dict(weight_decay=[0.1]), "weight decays"),
                        (dict(betas=(1.0, 0.9)), "betas"), (dict(state_bits=16), "state_bits"), (dict(max_norm=0.0), "max_norm"),
                        (dict(copies=[p[0].half(), p[1].bfloat16()]), "one half type"), (dict(copies=[None, p[0].half()]), "copy 1"), (dict(params=[p[0], p[0][1]], grads=[g[0], g[0][1]]), "share memory"),
                        (dict(params=[p[0], p[0]], grads=[g[0], g[0]]), "share memory")):
        with pytest.raises(ValueError, match=message):
            optim.AdamW(**{**dict(params=p, grads=g), **kw})


def test_dither_is_uniform():
    """The hash that rounds the 8-bit moments: both halves of its words are uniform and independent of each other and of the index --
    10^6 draws in 64 cells: chi-square with 63 degrees of freedom has mean 63 and deviation 11.2; six deviations allowed."""
    def draw(i, step, seed):
        h = (((i & 0xffffffff) ^ seed) + step * 0x9E3779B1 + (i >> 32) * 0xBB67AE85) & 0xffffffff
        h = ((h ^ (h >> 16)) * 0xBB67AE85) & 0xffffffff
        h = ((h ^ (h >> 15)) * 0x6A09E667) & 0xffffffff
        return h ^ (h >> 16)

    i = np.arange(1 << 20, dtype=np.uint64)
    for step, seed in ((1, 0), (2, 0), (1000, 7)):
        h = draw(i, np.uint64(step), np.uint64(seed)).astype(np.int64)
        later = draw(i, np.uint64(step + 1), np.uint64(seed)).astype(np.int64)
        for cell in (h >> 26, (h & 0xffff) >> 10, ((h >> 29) << 3) | ((h & 0xffff) >> 13), ((h >> 29) << 3) | (later >> 29), ((h[:-1] >> 29) << 3) | (h[1:] >> 29)):
            n = np.bincount(cell, minlength=64)
            expect = len(cell) / 64
            assert float(((n - expect) ** 2 / expect).sum()) < 63 + 6 * 11.2
