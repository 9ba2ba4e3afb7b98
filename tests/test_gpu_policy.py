"""GPU: scores, preference loss and clipped policy loss (csrc/policy_loss.hip) against their definitions in 64 bits.

Tolerances count roundings (u = 2^-24, one fp32 rounding; h = half a step of the logits' type):
  statistics  each e^(z - m) has the rounding of z - m and of its product with log2 e (each u |z - m|, weighted by softmax: D = sum p |z - m|)
              and 2 u of the exponential; a lane adds at most V / 256 + 32 terms, the joins 16: rs = u (2 + 3 D + V / 256 + 48)
  lp          rs + u (|z_t - m| + 2 |ln s| + |lp|): the two differences and the logarithm (2 u)
  p           rs + u (2 + 3 |z - m|) relative; the gradient c (1[t] - p) is rounded once to the logits' type (h relative, half of the least
              subnormal absolute), 4 u |c| for its products and the difference at the target
  c           the slope of dloss/dlp times the error of what it depends on, and 8 u relative for its own arithmetic
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


class Batch:
    """Logits of ragged sequences; lengths and how many leading rows of each are no action."""
    lanes = 256                                          # that add a row up

    def __init__(self, lengths, masked, vocab, dtype, seed=0, front=0, spare=0, pad=0, shift=0, spread=2.0):
        g = torch.Generator("cuda").manual_seed(seed)
        T = front + sum(lengths) + spare
        self.T, self.V, self.N, self.dtype = T, vocab, len(lengths), dtype
        # rows `vocab + pad` apart, starting `shift` elements behind an allocation's start
        flat = (torch.randn(T * (vocab + pad) + shift, device="cuda", generator=g) * spread).to(dtype)
        self.z = flat[shift:].view(T, vocab + pad)[:, :vocab]
        self.targets = torch.randint(0, vocab, (T,), device="cuda", generator=g, dtype=torch.int32)
        offs, live = [front], torch.zeros(T, dtype=torch.bool)
        for n, m in zip(lengths, masked):
            live[offs[-1] + m: offs[-1] + n] = True
            offs.append(offs[-1] + n)
        self.live = live.cuda()
        self.targets[~self.live] = -1
        if bool((~self.live).any()):
            self.z[~self.live] = math.nan                # what stands at masked positions is not looked at
        self.offs = torch.tensor(offs, dtype=torch.int32, device="cuda")
        self.g = g

    def rand(self, n, scale=1.0):
        return torch.randn(n, device="cuda", generator=self.g) * scale

    def reference(self):
        """lp, softmax, |z - m|, tolerance of lp, relative tolerance of the sum: 64 bits, masked rows zero."""
        z = torch.where(self.live.unsqueeze(1), self.z.double(), 0.0)
        m = z.amax(1, keepdim=True)
        d = (m - z).clamp(max=1e300)
        p = torch.softmax(z, 1)
        t = self.targets.clamp(min=0).long().unsqueeze(1)
        lp = torch.where(self.live, torch.log_softmax(z, 1).gather(1, t).squeeze(1), 0.0)
        rs = U * (2 + 3 * (p * d.clamp(max=1e30)).sum(1) + self.V / self.lanes + 48)
        lns = torch.logsumexp(z, 1) - m.squeeze(1)
        tol = rs + U * (d.gather(1, t).squeeze(1) + 2 * lns.abs() + lp.abs())
        return lp, p, d, torch.where(self.live, tol, 0.0), rs

    def sums(self, v):
        n = self.offs.long().tolist()
        return torch.stack([v[a:b].sum() for a, b in zip(n, n[1:])]) if self.N else v.new_zeros(0)

    def by_row(self, v, fill=0.0):
        out = torch.full((self.T,), fill, dtype=torch.float64, device="cuda")
        for k, (a, b) in enumerate(zip(self.offs.tolist(), self.offs.tolist()[1:])):
            out[a:b] = v[k]
        return out

    def gradient(self, c, dc, p, d, rs):
        """c (1[t] - p) and its tolerance, c with tolerance dc by row."""
        hot = torch.zeros_like(p).scatter_(1, self.targets.clamp(min=0).long().unsqueeze(1), 1.0)
        c, dc = torch.where(self.live, c, 0.0).unsqueeze(1), torch.where(self.live, dc, 0.0).unsqueeze(1)
        g = c * (hot - p)
        tol = (c.abs() * p * (rs.unsqueeze(1) + U * (2 + 3 * d.clamp(max=1e6))) + 4 * U * c.abs() * (hot + p) + dc * (hot - p).abs())
        half = torch.finfo(self.dtype).eps / 2
        return g, tol * (1 + half) + half * g.abs() + TINY[self.dtype] + 2.0 ** -149


def check(name, got, want, tol):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g times the tolerance" % (name, int(bad.sum()), bad.numel(), float(((got - want).abs() / tol).nan_to_num(math.inf).max()))


def new_gradient(b, pad=0, shift=0):
    flat = torch.full((b.T * (b.V + pad) + shift,), 7.0, dtype=b.dtype, device="cuda")
    return flat, flat[shift:].view(b.T, b.V + pad)[:, :b.V]


def untouched(b, flat, grad, pad, shift):
    """Rows of no sequence and everything between and behind the rows hold what was there."""
    own = torch.zeros_like(flat, dtype=torch.bool)
    view = own[shift:].view(b.T, b.V + pad)[:, :b.V]
    view[int(b.offs[0]): int(b.offs[-1])] = True
    assert bool((flat[~own] == 7.0).all())


def pair_reference(b, ref, w, beta, kind, margin, eps, norm, scale, gscale):
    lp, p, d, tol, rs = b.reference()
    n = b.sums(b.live.double()).clamp(min=1) if norm else torch.ones(b.N, dtype=torch.float64, device="cuda")
    LP, tLP = b.sums(lp) / n, b.sums(tol) / n
    # the result is rounded to fp32 once more
    diff = (LP - ref.double())[0::2] - (LP - ref.double())[1::2]
    tdiff = tLP[0::2] + tLP[1::2]
    if kind == "logistic":
        h = beta * diff - margin
        pair = (1 - eps) * torch.nn.functional.softplus(-h) + eps * torch.nn.functional.softplus(h)
        slope, curve, lip = beta * (torch.sigmoid(h) - (1 - eps)), beta * beta / 4, beta
    else:
        h = diff - 0.5 / beta
        pair, slope, curve, lip = h * h, 2 * h, 2.0, 2 * h.abs() + tdiff
    c = torch.stack((slope * w.double() * scale, -slope * w.double() * scale), 1).view(-1) / n * gscale
    dc = torch.stack((curve * tdiff * w.double() * scale,) * 2, 1).view(-1) / n * gscale + 8 * U * c.abs()
    g, tg = b.gradient(b.by_row(c), b.by_row(dc), p, d, rs)
    loss, tloss = (pair * w.double()).sum() * scale, ((lip * tdiff + 2 * U * pair) * w.double()).sum() * scale
    return dict(token=(lp, tol), seq=(LP, tLP + 2 * U * LP.abs()), diff=(diff, tdiff + 2 * U * diff.abs()),
                pair=(pair, lip * tdiff + 8 * U * pair), loss=(loss, tloss + 8 * U * loss.abs()), grad=(g, tg))


RAGGED = dict(lengths=[5, 3, 1, 7, 4, 0, 0, 2], masked=[2, 0, 0, 7, 1, 0, 0, 1])
# one item, odd sizes, word borders, every number of words a lane may hold
VOCABS = {"f32": [1, 2, 3, 5, 63, 1000, 1024, 1027, 4099, 16385, 65536, 70001], "f16": [1, 7, 9, 1001, 2049, 8191, 32771, 131075],
          "bf16": [1, 2, 15, 17, 1000, 2051, 8200, 32768, 131071, 140003]}
CASES = [(d, v) for d in VOCABS for v in VOCABS[d]]


@pytest.mark.parametrize("dtype,vocab", CASES)
def test_scores(dtype, vocab):
    from wide_deep_amd import policy
    b = Batch(vocab=vocab, dtype=DTYPES[dtype], seed=vocab, front=1, spare=2, **RAGGED)
    lp, _, _, tol, _ = b.reference()
    for norm in (False, True):
        r = policy.sequence_logp(b.z, b.targets, b.offs, length_norm=norm)
        n = b.sums(b.live.double()).clamp(min=1) if norm else 1.0
        check("token", r.token_logp, lp, tol)
        check("sequence", r.seq_logp, b.sums(lp) / n, b.sums(tol) / n + 2 * U * b.sums(lp).abs() / n)
        assert bool((r.token_logp[~b.live] == 0).all()) and bool((r.seq_logp[[3, 5, 6]] == 0).all())


@pytest.mark.parametrize("dtype,vocab", CASES)
@pytest.mark.parametrize("kind,norm", [("logistic", False), ("square", True)])
def test_preference_loss(dtype, vocab, kind, norm):
    from wide_deep_amd import policy
    b = Batch(vocab=vocab, dtype=DTYPES[dtype], seed=vocab + 1, front=2, spare=3, **RAGGED)
    ref, w = b.reference()[0], torch.rand(b.N // 2, device="cuda", generator=b.g) + 0.5
    ref = (b.sums(ref) * (0.3 if norm else 1.0) + b.rand(b.N, 3.0)).float()
    smooth, margin = (0.05, 0.25) if kind == "logistic" else (0.0, 0.0)
    gscale = 64.0
    want = pair_reference(b, ref, w, 0.1, kind, margin, smooth, norm, 0.25, gscale)
    flat, grad = new_gradient(b)
    r = policy.preference_loss(b.z, b.targets, b.offs, ref_logp=ref, weights=w, beta=0.1, kind=kind, margin=margin, label_smoothing=smooth,
                               length_norm=norm, reduction="mean", grad_scale=gscale, dlogits=grad)
    # beta, margin, smoothing and scale reach the kernel as fp32: 2^-24 relative of each
    for name, got in (("token", r.token_logp), ("seq", r.seq_logp), ("diff", r.difference), ("pair", r.pair_loss), ("loss", r.loss)):
        v, t = want[name]
        check(name, got, v, t + 16 * U * (v.abs() + (want["diff"][0].abs().max() + 5) * (name in ("pair", "loss"))))
    v, t = want["grad"]
    rows = slice(int(b.offs[0]), int(b.offs[-1]))
    check("gradient", grad[rows], v[rows], t[rows] + 16 * U * v[rows].abs().amax())
    untouched(b, flat, grad, 0, 0)


def policy_reference(b, old, adv_row, ref, clip, kl, reduction, gscale):
    lp, p, d, tol, rs = b.reference()
    count = b.sums(b.live.double())
    w = {"sum": torch.ones_like(lp), "token_mean": torch.ones_like(lp) / count.sum().clamp(min=1),
         "sequence_mean": b.by_row(1 / (count.clamp(min=1) * (count > 0).sum().clamp(min=1)))}[reduction]
    w = torch.where(b.live, w, 0.0)
    A = adv_row.double()
    x = torch.where(b.live, lp - old.double(), 0.0)
    rho = torch.exp(x)
    held = rho.clamp(1 - clip[0], 1 + clip[1])
    gone = rho * A > held * A
    loss, slope = -torch.minimum(rho * A, held * A), torch.where(gone, 0.0, -rho * A)
    k = torch.zeros_like(lp)
    lip, size = rho * A.abs(), rho * A.abs()
    if ref is not None:
        q = torch.where(b.live, ref.double() - lp, 0.0)
        k = torch.expm1(q) - q
        loss, slope = loss + kl * k, slope - kl * torch.expm1(q)
        lip = lip + kl * torch.expm1(q).abs() + kl * torch.exp(q) * tol
        size = size + kl * (torch.exp(q) + 1 + q.abs())
    te = tol + U * x.abs() + U * lp.abs()                       # error of an exponent
    tl = lip * te + 12 * U * size
    curve = rho * A.abs() + (kl * torch.exp(q) if ref is not None else 0.0)
    c, dc = slope * w * gscale, (curve * te + 12 * U * size) * w * gscale
    g, tg = b.gradient(c, dc, p, d, rs)
    tk = (torch.expm1(q).abs() + tol) * te + 12 * U * (torch.exp(q) + 1 + q.abs()) if ref is not None else torch.zeros_like(lp)
    s = lambda v, t: ((w * v).sum(), (w * (t + 4 * U * v.abs())).sum() + 2.0 ** -149)
    return dict(token=(lp, tol), loss=s(loss, tl), kl=s(k, tk), clipped=s((gone & b.live).double(), torch.zeros_like(lp)), grad=(g, tg))


@pytest.mark.parametrize("dtype,vocab", CASES)
@pytest.mark.parametrize("reduction,per_row,kl", [("sum", True, 0.0), ("token_mean", False, 0.1), ("sequence_mean", True, 0.1)])
def test_policy_loss(dtype, vocab, reduction, per_row, kl):
    from wide_deep_amd import policy
    b = Batch(vocab=vocab, dtype=DTYPES[dtype], seed=vocab + 2, front=1, spare=2, **RAGGED)
    lp = b.reference()[0]
    shift = b.rand(b.T, 0.2).double()
    for edge in (math.log1p(0.3), math.log1p(-0.2)):            # either side of a border is right next to it
        shift = torch.where((shift - edge).abs() < 1e-3, shift + 3e-3, shift)
    old, ref = (lp - shift).float(), (lp + b.rand(b.T, 0.3)).float() if kl else None
    adv = b.rand(b.T if per_row else b.N)
    gscale = 32.0
    want = policy_reference(b, old, adv if per_row else b.by_row(adv), ref, (0.2, 0.3), kl, reduction, gscale)
    flat, grad = new_gradient(b)
    r = policy.policy_loss(b.z, b.targets, b.offs, old, adv, ref_logp=ref, per_row=per_row, clip=(0.2, 0.3), kl_coef=kl, reduction=reduction,
                           grad_scale=gscale, dlogits=grad)
    for name, got in (("token", r.token_logp), ("loss", r.loss), ("kl", r.kl), ("clipped", r.clipped)):
        check(name, got, *want[name])
    v, t = want["grad"]
    rows = slice(int(b.offs[0]), int(b.offs[-1]))
    check("gradient", grad[rows], v[rows], t[rows])
    untouched(b, flat, grad, 0, 0)


def check_all(b, name=""):
    """Scores, both preference losses and the policy loss with every reduction against their definitions."""
    from wide_deep_amd import policy
    lp, _, _, tol, _ = b.reference()
    r = policy.sequence_logp(b.z, b.targets, b.offs)
    check(name + "token", r.token_logp, lp, tol)
    check(name + "sequence", r.seq_logp, b.sums(lp), b.sums(tol) + 2 * U * b.sums(lp).abs())
    rows = slice(int(b.offs[0]), int(b.offs[-1]))
    for kind, norm in (("logistic", False), ("square", True)):
        n = b.sums(b.live.double()).clamp(min=1) if norm else 1.0
        ref = (b.sums(lp) / n + b.rand(b.N, 2.0)).float()
        w = torch.rand(b.N // 2, device="cuda", generator=b.g) + 0.5
        want = pair_reference(b, ref, w, 0.1, kind, 0.0, 0.0, norm, 1.0, 16.0)
        r = policy.preference_loss(b.z, b.targets, b.offs, ref_logp=ref, weights=w, beta=0.1, kind=kind, length_norm=norm, grad_scale=16.0)
        for key, got in (("token", r.token_logp), ("seq", r.seq_logp), ("diff", r.difference), ("pair", r.pair_loss), ("loss", r.loss)):
            v, t = want[key]
            # beta, margin and scale reach the kernel as fp32: 2^-24 relative of each
            slack = 16 * U * (v.abs() + (want["diff"][0].abs().max() + 5) * (1.0 if key == "pair" else b.N if key == "loss" else 0.0))
            check("%s%s %s" % (name, kind, key), got, v, t + slack)
        v, t = want["grad"]
        check("%s%s gradient" % (name, kind), r.dlogits[rows], v[rows], t[rows] + 16 * U * v[rows].abs().amax())
        assert bool((r.dlogits[rows.stop:] == 0).all()) and bool((r.dlogits[:rows.start] == 0).all())
    for reduction, per_row, kl in (("sum", False, 0.1), ("token_mean", True, 0.0), ("sequence_mean", False, 0.1)):
        check_policy(b, reduction, per_row, kl, name)


def check_policy(b, reduction, per_row, kl, name=""):
    from wide_deep_amd import policy
    lp = b.reference()[0]
    shift = b.rand(b.T, 0.2).double()
    for edge in (math.log1p(0.3), math.log1p(-0.2)):
        shift = torch.where((shift - edge).abs() < 1e-3, shift + 3e-3, shift)
    old, ref = (lp - shift).float(), (lp + b.rand(b.T, 0.3)).float() if kl else None
    adv = b.rand(b.T if per_row else b.N)
    want = policy_reference(b, old, adv if per_row else b.by_row(adv), ref, (0.2, 0.3), kl, reduction, 32.0)
    r = policy.policy_loss(b.z, b.targets, b.offs, old, adv, ref_logp=ref, per_row=per_row, clip=(0.2, 0.3), kl_coef=kl, reduction=reduction, grad_scale=32.0)
    for key, got in (("token", r.token_logp), ("loss", r.loss), ("kl", r.kl), ("clipped", r.clipped)):
        check("%s%s %s" % (name, reduction, key), got, *want[key])
    rows = slice(int(b.offs[0]), int(b.offs[-1]))
    check("%s%s gradient" % (name, reduction), r.dlogits[rows], want["grad"][0][rows], want["grad"][1][rows])
    assert bool((r.dlogits[rows.stop:] == 0).all())


@pytest.mark.parametrize("rows,seqs,vocab,dtype", [(70, 6, 2048, "f32"), (70, 6, 4096, "bf16"), (66, 64, 900, "f16"), (300, 10, 8193, "f32"), (300, 30, 33001, "bf16"),
                                                   (257, 258, 700, "bf16"), (2100, 12, 301, "f16"), (2100, 40, 9001, "bf16"), (5000, 1600, 37, "f32"), (70000, 1200, 5, "f16")])
def test_ways_of_the_kernels(rows, seqs, vocab, dtype):
    """Batches on either side of the limits at which the launches change: rows and sequences that are many or few, rows short or split."""
    g = torch.Generator().manual_seed(rows + seqs)
    seqs += seqs % 2
    share = torch.rand(seqs, generator=g) * (torch.rand(seqs, generator=g) < 0.9)
    lengths = (share / share.sum() * rows).floor().int().tolist()
    masked = [n if k % 7 == 3 else n // 4 for k, n in enumerate(lengths)]
    check_all(Batch(lengths, masked, vocab, DTYPES[dtype], seed=rows, front=1, spare=rows - sum(lengths) - 1))


@pytest.mark.parametrize("words", [1, 65, 128, 129, 257, 400, 513, 1100, 2048, 2049, 3100, 4097, 4700, 5200, 5700, 6200, 6700, 7200, 8200, 9300, 10300, 11300, 12800,
                                   12801, 14400, 16384, 16385])
def test_policy_rows_of_every_register_count(words):
    """One row length for each number of 16-byte words a lane may hold, and its neighbours at the limits."""
    check_policy(Batch([3, 2], [1, 0], 8 * words + 3, torch.bfloat16, seed=words), "sequence_mean", False, 0.1)
    check_policy(Batch([2, 200, 100], [1, 0, 50], 8 * words - 1, torch.bfloat16, seed=words), "token_mean", True, 0.0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("pad,shift,gpad,gshift", [(0, 1, 0, 1), (3, 0, 3, 0), (5, 3, 0, 0), (0, 0, 1, 2), (8, 0, 8, 4)])
def test_strides_and_alignments(dtype, pad, shift, gpad, gshift):
    """Rows that start anywhere, gradients that start elsewhere; nothing between the rows is written."""
    from wide_deep_amd import policy
    for vocab in (5, 301, 9001, 140001):
        b = Batch([4, 3], [1, 0], vocab, DTYPES[dtype], seed=3, spare=1, pad=pad, shift=shift)
        plain = Batch([4, 3], [1, 0], vocab, DTYPES[dtype], seed=3, spare=1)
        plain.z, b_z = b.z.contiguous(), b.z
        adv, old = b.rand(b.T), torch.where(b.live, b.reference()[0], 0.0).float() - 0.05
        for call in (lambda z, g: policy.preference_loss(z, b.targets, b.offs, dlogits=g),
                     lambda z, g: policy.policy_loss(z, b.targets, b.offs, old, adv, dlogits=g)):
            flat, grad = new_gradient(b, gpad, gshift)
            r, q = call(b_z, grad), call(plain.z, True)
            untouched(b, flat, grad, gpad, gshift)
            _, p, d, _, rs = b.reference()
            end = int(b.offs[-1])
            # the same numbers added in another order: twice the tolerance of the definition
            c = q.dlogits.double().abs().amax()
            check("token", r.token_logp, q.token_logp, 2 * b.reference()[3] + 1e-30)
            check("gradient", grad[:end], q.dlogits[:end], 2 * (torch.finfo(b.dtype).eps + rs.max() + 60 * U) * q.dlogits[:end].double().abs() + 64 * U * c + TINY[b.dtype] * 2)
            assert bool((q.dlogits[end:] == 0).all())


def test_masks_infinities_and_lowest_values():
    """-inf items have probability 0; a row at the type's lowest value is uniform; what is undefined stays in its own row and pair."""
    from wide_deep_amd import policy
    for dtype in DTYPES.values():
        for V in (40, 3001, 140001):
            low = torch.finfo(dtype).min
            b = Batch([2, 2, 2, 2], [0, 0, 0, 0], V, dtype, seed=9)
            z = b.z
            z[0, 1:] = -math.inf                                  # one item left
            b.targets[0] = 0
            z[1, ::2] = -math.inf
            b.targets[1] = 1
            z[2] = low                                            # uniform
            z[3, 5:] = low
            b.targets[3] = 2
            z[4] = -math.inf                                      # no distribution at all: NaN, in this pair only
            z[6, 0] = math.inf
            adv = torch.ones(4, device="cuda")
            r = policy.sequence_logp(z, b.targets, b.offs)
            want = torch.log_softmax(z.double(), 1).gather(1, b.targets.long().unsqueeze(1)).squeeze(1)
            good = torch.tensor([0, 1, 2, 3, 5, 7], device="cuda")
            # rows as in the definition; |z - m| of the lowest value counts nothing, its weight is 0
            check("token", r.token_logp[good], want[good], U * (100 + V / 256 + 8 * want[good].abs()))
            assert float(r.token_logp[0]) == 0.0 and bool(r.token_logp[[4, 6]].isnan().all())
            for q in (policy.preference_loss(z, b.targets, b.offs), policy.policy_loss(z, b.targets, b.offs, r.token_logp.nan_to_num(0.0), adv)):
                assert bool(q.dlogits[:4].isfinite().all()) and bool((q.dlogits[1, ::2] == 0).all())
                assert bool(q.dlogits[4].isnan().all()) and bool((q.dlogits[0].abs() == 0).all())
            # an item that cannot be chosen was: its log-probability is -inf, the slope of its pair stays finite
            t = b.targets.clone()
            t[1] = 0
            q = policy.preference_loss(z[:4], t[:4], b.offs[:3])
            assert float(q.token_logp[1]) == -math.inf and float(q.difference[0]) == -math.inf and bool(q.dlogits.isfinite().all())
            assert float(q.pair_loss[0]) == math.inf


@pytest.mark.parametrize("rows,seqs,vocab,dtype", [(900, 12, 5000, "bf16"), (900, 70, 3001, "f16"), (1024, 64, 600, "f32"), (1030, 64, 600, "f32"), (30, 5, 70001, "f32"), (280, 9, 140003, "f16"),
                                                   (600, 3, 66001, "f32"), (2500, 256, 333, "bf16"), (2500, 258, 333, "bf16")])
@pytest.mark.parametrize("reduction", ["sum", "token_mean", "sequence_mean"])
def test_weights_that_rows_find_themselves(rows, seqs, vocab, dtype, reduction):
    """Both sides of the sizes up to which a policy loss needs no launch for weights, rows in registers and rows too long for them."""
    g = torch.Generator().manual_seed(rows)
    share = torch.rand(seqs, generator=g) * (torch.rand(seqs, generator=g) < 0.8)
    share[0] = 1.0
    lengths = (share / share.sum() * (rows - 3)).floor().int().tolist()
    masked = [n if k % 5 == 4 else n // 3 for k, n in enumerate(lengths)]
    b = Batch(lengths, masked, vocab, DTYPES[dtype], seed=seqs, front=2, spare=rows - 2 - sum(lengths))
    check_policy(b, reduction, False, 0.1)
    check_policy(b, reduction, True, 0.0)
    if vocab > 60000:                                            # the loss alone, and a gradient in the logits' place
        from wide_deep_amd import policy
        old, adv = b.reference()[0].float(), b.rand(b.N)
        want = policy.policy_loss(b.z, b.targets, b.offs, old, adv, per_row=False, reduction=reduction)
        alone = policy.policy_loss(b.z, b.targets, b.offs, old, adv, per_row=False, reduction=reduction, dlogits=None)
        z = b.z.clone()
        place = policy.policy_loss(z, b.targets, b.offs, old, adv, per_row=False, reduction=reduction, dlogits=z)
        first, last = int(b.offs[0]), int(b.offs[-1])
        for r in (alone, place):
            assert torch.equal(r.loss, want.loss) and torch.equal(r.token_logp, want.token_logp)
        assert torch.equal(z[first:last], want.dlogits[first:last])


@pytest.mark.parametrize("rows,seqs,vocab,dtype", [(1024, 64, 300, "bf16"), (1025, 64, 300, "bf16"), (1024, 66, 300, "f16"), (2048, 6, 16390, "bf16"), (2049, 6, 16390, "bf16"), (2048, 2, 8193, "f32"),
                                                   (1024, 2, 700, "f32"), (200, 64, 900, "f32"), (200, 128, 900, "f32")])
def test_pairs_that_rows_find_themselves(rows, seqs, vocab, dtype):
    """Both sides of the sizes up to which a preference loss needs no launch for its pairs: empty sequences, and pairs as long as the batch."""
    from wide_deep_amd import policy
    g = torch.Generator().manual_seed(rows)
    share = torch.rand(seqs, generator=g) * (torch.rand(seqs, generator=g) < 0.8)
    share[0] = 1.0
    lengths = (share / share.sum() * (rows - 3)).floor().int().tolist()
    masked = [n if k % 5 == 4 else n // 3 for k, n in enumerate(lengths)]
    b = Batch(lengths, masked, vocab, DTYPES[dtype], seed=seqs, front=2, spare=rows - 2 - sum(lengths))
    ref, w = b.rand(seqs, 3.0), torch.rand(seqs // 2, device="cuda", generator=b.g) + 0.5
    for kind, norm in (("logistic", False), ("logistic", True), ("square", True)):
        n = b.sums(b.live.double()).clamp(min=1) if norm else 1.0
        near = (b.sums(b.reference()[0]) / n).float() + ref
        want = pair_reference(b, near, w, 0.1, kind, 0.0, 0.0, norm, 1.0, 16.0)
        r = policy.preference_loss(b.z, b.targets, b.offs, ref_logp=near, weights=w, beta=0.1, kind=kind, length_norm=norm, grad_scale=16.0)
        for key, got in (("token", r.token_logp), ("seq", r.seq_logp), ("diff", r.difference), ("pair", r.pair_loss), ("loss", r.loss)):
            v, t = want[key]
            # beta, margin and scale reach the kernel as fp32: 2^-24 relative of each
            slack = 16 * U * (v.abs() + (want["diff"][0].abs().max() + 5) * (1.0 if key == "pair" else b.N if key == "loss" else 0.0))
            check("%s %s" % (kind, key), got, v, t + slack)
        v, t = want["grad"]
        own = slice(int(b.offs[0]), int(b.offs[-1]))
        check("%s gradient" % kind, r.dlogits[own], v[own], t[own] + 16 * U * v[own].abs().amax())


def test_kl_that_is_only_told():
    """kl_coef 0 with ref_logp: k is reported, and an infinite one (a reference that has not got the item's probability down) moves nothing."""
    from wide_deep_amd import policy
    for seqs in (1, 40):                                         # one launch, and weights from launches of their own
        b = Batch([9] * seqs, [0] * seqs, 700, torch.float32, seed=seqs)
        old, adv = policy.sequence_logp(b.z, b.targets, b.offs).token_logp + 0.1, b.rand(seqs)
        ref = old.clone()
        ref[3] = 200.0                                           # e^200 is beyond fp32
        with_ref = policy.policy_loss(b.z, b.targets, b.offs, old, adv, ref)
        without = policy.policy_loss(b.z, b.targets, b.offs, old, adv)
        assert float(with_ref.kl) == math.inf and float(without.kl) == 0.0
        assert torch.equal(with_ref.loss, without.loss) and torch.equal(with_ref.dlogits, without.dlogits) and bool(without.dlogits.isfinite().all())


@pytest.mark.parametrize("rows,words", [(1, 2048), (1, 2049), (2, 4096), (3, 4097), (1, 8192), (1, 16384)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_few_rows_that_are_long(rows, words, dtype):
    """Both sides of the lengths at which a handful of rows goes to one workgroup."""
    b = Batch([1, rows - 1], [0, 0], words * (4 if dtype == "f32" else 8), DTYPES[dtype], seed=words)
    b.lanes = 64                                                 # a wavefront adds a row up
    check_all(b)


def test_empty_calls_and_refusals():
    from wide_deep_amd import capi, policy
    i32 = dict(dtype=torch.int32, device="cuda")
    z = torch.randn(3, 10, device="cuda")
    none, nothing = torch.zeros(1, **i32), torch.full((3,), -1, **i32)
    r = policy.sequence_logp(z, torch.zeros(3, **i32), none)                             # no sequence: every row belongs to nobody
    assert r.token_logp.tolist() == [0, 0, 0] and r.seq_logp.numel() == 0
    q = policy.preference_loss(z, torch.zeros(3, **i32), none)
    assert float(q.loss) == 0.0 and bool((q.dlogits == 0).all())
    q = policy.policy_loss(z, torch.zeros(3, **i32), none, torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda"))
    assert float(q.loss) == 0.0 and bool((q.dlogits == 0).all())
    two = torch.tensor([0, 1, 3], **i32)
    q = policy.preference_loss(z, nothing, two, beta=0.5)                                # no action: log 2 and no gradient
    assert abs(float(q.loss) - math.log(2)) < 1e-6 and bool((q.dlogits == 0).all()) and q.seq_logp.tolist() == [0, 0]
    q = policy.policy_loss(z, nothing, two, torch.zeros(3, device="cuda"), torch.ones(2, device="cuda"), reduction="sequence_mean")
    assert float(q.loss) == 0.0 and bool((q.dlogits == 0).all())
    empty = torch.empty(0, 10, device="cuda")
    q = policy.preference_loss(empty, torch.zeros(0, **i32), torch.zeros(3, **i32), dlogits=None)
    assert abs(float(q.loss) - math.log(2)) < 1e-6 and q.dlogits is None
    q = policy.policy_loss(empty, torch.zeros(0, **i32), torch.zeros(3, **i32), empty[:, 0], torch.ones(2, device="cuda"))
    assert float(q.loss) == 0.0 and q.dlogits.shape == (0, 10)
    far = torch.tensor([10, 7, -5], **i32)                                               # items that do not exist are no actions
    assert policy.sequence_logp(z, far, two).token_logp[[0, 2]].tolist() == [0, 0]
    # offsets outside the rows are cut to them
    assert bool(policy.sequence_logp(z, torch.zeros(3, **i32), torch.tensor([-4, 1, 90], **i32)).token_logp.isfinite().all())
    t = torch.zeros(3, **i32)
    for bad in (lambda: policy.sequence_logp(z, t[:2], two), lambda: policy.sequence_logp(z, t.long(), two), lambda: policy.sequence_logp(z, t.cpu(), two),
                lambda: policy.sequence_logp(z, t, two.long()), lambda: policy.preference_loss(z, t, two[:2]),
                lambda: policy.preference_loss(z, t, two, ref_logp=torch.zeros(3, device="cuda")), lambda: policy.preference_loss(z, t, two, kind="cube"),
                lambda: policy.preference_loss(z, t, two, reduction="max"), lambda: policy.preference_loss(z, t, two, weights=torch.ones(2, device="cuda")),
                lambda: policy.preference_loss(z, t, two, dlogits=z.half()), lambda: policy.preference_loss(z, t, two, dlogits=z[:2]),
                lambda: policy.policy_loss(z, t, two, torch.zeros(2, device="cuda"), torch.ones(2, device="cuda")),
                lambda: policy.policy_loss(z, t, two, torch.zeros(3, device="cuda"), torch.ones(4, device="cuda")),
                lambda: policy.policy_loss(z, t, two, torch.zeros(3, device="cuda"), torch.ones(2, device="cuda"), kl_coef=0.1),
                lambda: policy.policy_loss(z, t, torch.arange(4, **i32), torch.zeros(3, device="cuda"), torch.ones(3, device="cuda")),
                lambda: policy.policy_loss(z, t, two, torch.zeros(3, device="cuda"), torch.ones(2, device="cuda"), reduction="mean")):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(capi.WdError, match="clip range"):
        policy.policy_loss(z, t, two, torch.zeros(3, device="cuda"), torch.ones(2, device="cuda"), clip=(-0.1, 0.2))
    with pytest.raises(capi.WdError, match="beta"):
        policy.preference_loss(z, t, two, beta=0.0)


def test_gradients_against_differences():
    """dlogits against central differences of the definitions' losses: step 1e-5 in 64 bits is off by 1e-10 and 1e-11 of rounding."""
    from wide_deep_amd import policy
    b = Batch([3, 2, 4, 1], [1, 0, 0, 0], 23, torch.float32, seed=5, spread=1.0)
    w = torch.tensor([0.7, 1.3], device="cuda")
    old, ref, adv = b.reference()[0].float() - 0.05, b.reference()[0].float() + 0.2, b.rand(b.N)
    cases = [(lambda: policy.preference_loss(b.z, b.targets, b.offs, weights=w, beta=0.4).dlogits,
              lambda: pair_reference(b, torch.zeros(4, device="cuda"), w, 0.4, "logistic", 0.0, 0.0, False, 1.0, 1.0)["loss"][0]),
             (lambda: policy.preference_loss(b.z, b.targets, b.offs, weights=w, beta=0.4, kind="square", length_norm=True).dlogits,
              lambda: pair_reference(b, torch.zeros(4, device="cuda"), w, 0.4, "square", 0.0, 0.0, True, 1.0, 1.0)["loss"][0]),
             (lambda: policy.policy_loss(b.z, b.targets, b.offs, old, adv, ref_logp=ref, kl_coef=0.3, reduction="sequence_mean").dlogits,
              lambda: policy_reference(b, old, b.by_row(adv), ref, (0.2, 0.2), 0.3, "sequence_mean", 1.0)["loss"][0])]
    for kernel, loss in cases:
        grad, z = kernel(), b.z
        for r, v in ((1, 0), (1, int(b.targets[1])), (2, 22), (4, 7), (6, int(b.targets[6])), (9, 3)):
            b.z = z.double()
            b.z[r, v] += 1e-5
            up = loss()
            b.z[r, v] -= 2e-5
            down = loss()
            b.z = z
            # 2^-23 of the largest coefficient for the fp32 kernel, as everywhere above
            assert abs(float(grad[r, v]) - float((up - down) / 2e-5)) < 1e-8 + 64 * U * float(grad.abs().max())


def test_streams_graphs_and_shared_buffers():
    """The same bits on another stream, two calls at once, from a replayed graph beside the program's own calls, and in place."""
    from wide_deep_amd import hipgraph, policy
    b = Batch([30, 20, 9, 40], [3, 0, 1, 10], 5003, torch.bfloat16, seed=4)
    c = Batch([11, 60, 2, 1], [3, 0, 1, 0], 5003, torch.bfloat16, seed=6)
    old = {id(x): x.reference()[0].float() - 0.1 for x in (b, c)}
    adv = b.rand(4)

    def both(x):
        p = policy.preference_loss(x.z, x.targets, x.offs)
        q = policy.policy_loss(x.z, x.targets, x.offs, old[id(x)], adv)
        return [v for r in (p, q, policy.sequence_logp(x.z, x.targets, x.offs)) for v in r]

    same = lambda a, w: all(torch.equal(x.nan_to_num(), y.nan_to_num()) for x, y in zip(a, w))
    want, want_c = both(b), both(c)
    assert same(both(b), want)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(s1):
            x = both(b)
        with torch.cuda.stream(s2):
            y = both(c)
    torch.cuda.synchronize()
    assert same(x, want) and same(y, want_c)
    graphs = []
    for x in (b, c):
        with torch.cuda.stream(s1):
            both(x)
        torch.cuda.synchronize()
        g = hipgraph.new_graph()
        with torch.cuda.graph(g, stream=s1):
            out = both(x)
        graphs.append((g, out))
    for _ in range(3):
        for (g, out), w in zip(graphs, (want, want_c)):
            for v in out:
                v.zero_()
            g.replay()
            eager = both(c)
            torch.cuda.synchronize()
            assert same(out, w) and same(eager, want_c)
    z = b.z.clone()
    r = policy.preference_loss(z, b.targets, b.offs, dlogits=z)
    assert same(r, want[:6]) and r.dlogits is z
    z = b.z.clone()
    assert same(policy.policy_loss(z, b.targets, b.offs, old[id(b)], adv, dlogits=z), want[6:11])


@pytest.mark.parametrize("rows,vocab,dtype", [(400, 9001, "bf16"), (90, 60001, "f32"), (9, 300001, "bf16"), (600, 20001, "f16"), (3000, 501, "f32"), (40, 200, "f32")])
def test_gradient_in_the_place_of_the_logits(rows, vocab, dtype):
    """The same bits whether the gradient has a buffer of its own or the logits': no launch reads a logit that another row's may overwrite."""
    from wide_deep_amd import policy
    n = rows // 4
    b = Batch([n, n, n, rows - 3 * n], [1, 0, n // 2, 0], vocab, DTYPES[dtype], seed=rows)
    old, adv = b.reference()[0].float() - 0.1, b.rand(4)
    for call in (lambda z, g: policy.preference_loss(z, b.targets, b.offs, dlogits=g), lambda z, g: policy.policy_loss(z, b.targets, b.offs, old, adv, per_row=False, dlogits=g)):
        want = call(b.z, True)
        for _ in range(8):
            z = b.z.clone()
            got = call(z, z)
            assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_offsets_past_32_bits():
    """A row that starts behind 2^32 elements."""
    from wide_deep_amd import policy
    V, T = 70001, 65000
    z = torch.empty(T, V, dtype=torch.bfloat16, device="cuda")
    b = Batch([2, 2], [0, 0], V, torch.bfloat16, seed=2)
    t = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    rows = torch.tensor([0, 5, T - 2, T - 1], device="cuda")
    z[rows], t[rows] = b.z, b.targets
    offs = torch.tensor([0, 6, T], dtype=torch.int32, device="cuda")
    small = policy.preference_loss(b.z, b.targets, b.offs)
    large = policy.preference_loss(z, t, offs, dlogits=z)
    assert torch.equal(large.seq_logp, small.seq_logp)
    check("gradient", z[rows], small.dlogits, small.dlogits.double().abs() * torch.finfo(torch.bfloat16).eps + 1e-30)
    assert bool((z[6: 2000] == 0).all())
