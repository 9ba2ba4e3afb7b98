"""GPU: what the policy heads answer where a log-probability, a ratio or a difference is infinite (csrc/policy_loss.hip), and losses without a
gradient, each in every way that the launches take."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# rows, vocab, type: a handful in one launch, short rows, rows split over workgroups, many sequences, rows longer than the registers
SHAPES = [(8, 100, "f32"), (400, 300, "bf16"), (40, 9001, "f32"), (3000, 501, "f16"), (2600, 40, "f32"), (40, 140003, "bf16"), (1500, 66001, "f32")]
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(rows, vocab, dtype, seqs=4, seed=0):
    """Logits, targets, offsets of `seqs` sequences of equal length; row 1 of the second sequence has an item that cannot be chosen, and it was."""
    g = torch.Generator("cuda").manual_seed(rows + vocab + seed)
    z = torch.randn(rows, vocab, device="cuda", generator=g).to(DTYPES[dtype])
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g, dtype=torch.int32)
    per = rows // seqs
    offs = torch.arange(seqs + 1, device="cuda", dtype=torch.int32) * per
    bad = per + 1
    z[bad, int(t[bad])] = -math.inf
    return z, t, offs, bad


def several(rows):
    return 4 if rows < 2600 else 4 if rows == 3000 else 1300


@pytest.mark.parametrize("rows,vocab,dtype", SHAPES)
@pytest.mark.parametrize("norm", [False, True])
def test_a_rejected_sequence_that_cannot_be(rows, vocab, dtype, norm):
    """d = +inf: the pair is settled, its loss is 0 (label_smoothing 0) and it moves nothing; with smoothing the loss is +inf, the slope beta eps."""
    from wide_deep_amd import policy
    z, t, offs, bad = make(rows, vocab, dtype, several(rows))
    a, b, c = offs[:3].tolist()
    w = torch.full((len(offs) // 2,), 0.5, device="cuda")
    for margin in (0.0, 0.25):
        r = policy.preference_loss(z, t, offs, weights=w, margin=margin, length_norm=norm)
        assert float(r.token_logp[bad]) == -math.inf and float(r.seq_logp[1]) == -math.inf and float(r.difference[0]) == math.inf
        assert float(r.pair_loss[0]) == 0.0 and bool(r.pair_loss.isfinite().all())
        want = float((r.pair_loss.double() * 0.5).sum())
        assert abs(float(r.loss) - want) <= 2.0 ** -22 * want + 2.0 ** -24 * float(r.pair_loss.double().sum())      # pair_loss and loss round once each
        assert bool((r.dlogits[a:c] == 0).all()) and bool(r.dlogits.isfinite().all()) and bool((r.dlogits[c:] != 0).any())
    smooth = policy.preference_loss(z, t, offs, label_smoothing=0.1, length_norm=norm)
    assert float(smooth.pair_loss[0]) == math.inf and float(smooth.loss) == math.inf and bool(smooth.dlogits.isfinite().all())
    # the other way round: the chosen one cannot be
    t2 = t.clone()
    z2 = z.clone()
    z2[bad] = z[bad].nan_to_num(0.0, neginf=0.0)
    z2[1, int(t[1])] = -math.inf
    r = policy.preference_loss(z2, t2, offs, length_norm=norm)
    assert float(r.difference[0]) == -math.inf and float(r.pair_loss[0]) == math.inf and bool(r.dlogits.isfinite().all())


@pytest.mark.parametrize("rows,vocab,dtype", SHAPES)
@pytest.mark.parametrize("reduction", ["sum", "token_mean", "sequence_mean"])
def test_kl_of_an_item_that_cannot_be(rows, vocab, dtype, reduction):
    """token_logp = -inf under a reference that could choose the item: k = e^inf - inf - 1 = +inf; with kl_coef 0 it is told and moves nothing."""
    from wide_deep_amd import policy
    z, t, offs, bad = make(rows, vocab, dtype, several(rows))
    ref = policy.sequence_logp(z, t, offs).token_logp.clone()
    assert float(ref[bad]) == -math.inf
    ref[bad] = -3.0
    adv = torch.ones(len(offs) - 1, device="cuda")
    call = lambda **kw: policy.policy_loss(z, t, offs, ref, adv, per_row=False, reduction=reduction, **kw)
    told, without, alone = call(ref_logp=ref), call(), call(ref_logp=ref, dlogits=None)
    for r in (told, alone):
        assert float(r.kl) == math.inf and torch.equal(r.loss, without.loss) and bool(r.loss.isfinite())
    assert torch.equal(told.dlogits, without.dlogits) and bool(told.dlogits.isfinite().all()) and bool((told.dlogits[bad] == 0).all())
    taken = call(ref_logp=ref, kl_coef=0.1)
    others = torch.arange(rows, device="cuda") != bad
    assert float(taken.kl) == math.inf and float(taken.loss) == math.inf and bool(taken.dlogits[others].isfinite().all())
    # a reference that could not choose the item either side of it: k = e^-inf + inf - 1
    far = ref.clone()
    far[bad + 1] = -math.inf
    z2 = z.clone()
    z2[bad] = z[bad].nan_to_num(0.0, neginf=0.0)
    r = policy.policy_loss(z2, t, offs, ref, adv, ref_logp=far, per_row=False, reduction=reduction, kl_coef=0.1)
    assert float(r.kl) == math.inf and float(r.loss) == math.inf and bool(r.dlogits.isfinite().all())


@pytest.mark.parametrize("rows,vocab,dtype", SHAPES)
@pytest.mark.parametrize("clip", [(0.2, 0.2), (1.0, math.inf)])
def test_an_advantage_of_zero_tells_nothing_whatever_the_ratio(rows, vocab, dtype, clip):
    """rho = e^(lp - old) above fp32 (old far below, or -inf): 0 x inf is no loss and no slope.  With another advantage it stays what it was."""
    from wide_deep_amd import policy
    z, t, offs, bad = make(rows, vocab, dtype, several(rows))
    z[bad] = z[bad].nan_to_num(0.0, neginf=0.0)
    lp = policy.sequence_logp(z, t, offs).token_logp
    old, adv = lp - 0.05, torch.ones(rows, device="cuda")
    for far in (lp[1] - 100.0, torch.tensor(-math.inf)):
        old[1], adv[1] = far, 0.0
        for zero in (0.0, -0.0):
            adv[1] = zero
            r = policy.policy_loss(z, t, offs, old, adv, per_row=True, clip=clip, reduction="sum")
            near = old.clone()
            near[1] = lp[1]
            want = policy.policy_loss(z, t, offs, near, adv, per_row=True, clip=clip, reduction="sum")
            assert torch.equal(r.loss, want.loss) and torch.equal(r.clipped, want.clipped) and bool((r.dlogits[1] == 0).all())
            assert torch.equal(r.dlogits, want.dlogits)
            alone = policy.policy_loss(z, t, offs, old, adv, per_row=True, clip=clip, reduction="sum", dlogits=None)
            assert torch.equal(alone.loss, want.loss)
        adv[1] = -1.0
        r = policy.policy_loss(z, t, offs, old, adv, per_row=True, clip=clip, reduction="sum")
        assert float(r.loss) == math.inf
        if clip[1] < 1.0:
            adv[1] = 1.0
            r = policy.policy_loss(z, t, offs, old, adv, per_row=True, clip=clip, reduction="sum")
            assert bool(r.loss.isfinite()) and bool((r.dlogits[1] == 0).all()) and float(r.clipped) == 1.0


@pytest.mark.parametrize("rows,vocab,dtype", SHAPES)
@pytest.mark.parametrize("kind", ["logistic", "square"])
def test_pairs_of_weight_zero_add_nothing(rows, vocab, dtype, kind):
    """A pair left out by its weight is left out, an infinite loss of its own is told in pair_loss and nowhere else."""
    from wide_deep_amd import policy
    z, t, offs, bad = make(rows, vocab, dtype, several(rows))
    a, b, c = offs[:3].tolist()
    z[bad] = z[bad].nan_to_num(0.0, neginf=0.0)
    z[1, int(t[1])] = -math.inf                              # the chosen sequence of the first pair cannot be
    w = torch.full((len(offs) // 2,), 0.5, device="cuda")
    w[0] = 0.0
    r = policy.preference_loss(z, t, offs, weights=w, kind=kind)
    assert float(r.difference[0]) == -math.inf and float(r.pair_loss[0]) == math.inf
    want = float((r.pair_loss[1:].double() * 0.5).sum())
    assert abs(float(r.loss) - want) <= 2.0 ** -23 * want      # pair_loss and loss round once each
    assert bool((r.dlogits[a:c] == 0).all()) and bool(r.dlogits.isfinite().all()) and bool((r.dlogits[c:] != 0).any())


def test_gradients_beside_the_logits_rows():
    """Logits and gradient as halves of one buffer's rows are apart; places that share memory with the logits without being theirs are refused."""
    from wide_deep_amd import capi, policy
    for rows, vocab in ((8, 40), (300, 1001), (12, 70001)):
        g = torch.Generator("cuda").manual_seed(rows)
        both = torch.randn(rows, 2 * vocab, device="cuda", generator=g)
        z, place = both[:, :vocab], both[:, vocab:]
        t = torch.randint(0, vocab, (rows,), device="cuda", generator=g, dtype=torch.int32)
        offs = torch.tensor([0, rows // 4, rows // 2, rows - 1, rows], device="cuda", dtype=torch.int32)
        adv, old = torch.randn(4, device="cuda", generator=g), policy.sequence_logp(z, t, offs).token_logp - 0.1
        for call in (lambda g: policy.preference_loss(z, t, offs, dlogits=g), lambda g: policy.policy_loss(z, t, offs, old, adv, per_row=False, dlogits=g)):
            was = z.clone()
            want = call(True).dlogits
            got = call(place)
            assert got.dlogits is place and torch.equal(place, want) and torch.equal(z, was)
            for bad in (both[:, 1: vocab + 1], both[:, vocab - 1: 2 * vocab - 1]):
                with pytest.raises(capi.WdError, match="shares memory"):
                    call(bad)
            assert torch.equal(z, was)


@pytest.mark.parametrize("rows,vocab,dtype", SHAPES + [(1, 7, "f16"), (64, 1000, "bf16"), (1024, 64, "f32"), (5, 70001, "f32")])
def test_losses_without_a_gradient(rows, vocab, dtype):
    """dlogits None: the same bits as beside a gradient, and nothing else is written."""
    from wide_deep_amd import policy
    g = torch.Generator("cuda").manual_seed(rows)
    z = torch.randn(rows, vocab, device="cuda", generator=g).to(DTYPES[dtype])
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g, dtype=torch.int32)
    t[rows // 3] = -1
    cuts = sorted({0, rows // 5, rows // 2, rows // 2 + 1, rows} & set(range(rows + 1)))
    offs = torch.tensor(cuts + [rows] * (5 - len(cuts)), dtype=torch.int32, device="cuda")
    was = z.clone()
    ref = torch.randn(4, device="cuda", generator=g)
    for kw in (dict(), dict(kind="square", length_norm=True, reduction="mean"), dict(margin=0.3, label_smoothing=0.1, weights=torch.rand(2, device="cuda", generator=g))):
        full = policy.preference_loss(z, t, offs, ref_logp=ref, **kw)
        for none in (None, False):
            alone = policy.preference_loss(z, t, offs, ref_logp=ref, dlogits=none, **kw)
            assert alone.dlogits is None and all(torch.equal(x, y) for x, y in zip(alone[:5], full[:5])) and bool(full.loss.isfinite())
    old = policy.sequence_logp(z, t, offs).token_logp + torch.randn(rows, device="cuda", generator=g) * 0.1
    adv = torch.randn(4, device="cuda", generator=g)
    for kw in (dict(reduction="sum"), dict(reduction="token_mean", ref_logp=old, kl_coef=0.1), dict(reduction="sequence_mean")):
        full = policy.policy_loss(z, t, offs, old, adv, per_row=False, **kw)
        alone = policy.policy_loss(z, t, offs, old, adv, per_row=False, dlogits=None, **kw)
        assert alone.dlogits is None and all(torch.equal(x, y) for x, y in zip(alone[:4], full[:4])) and bool(full.loss.isfinite())
    assert torch.equal(z, was)
