"""GPU: AdamW over many tensors (csrc/adamw.hip) against its formula in 64 bits; u = 2^-24, one fp32 rounding.

  m, v     two products and a sum, constants and the clipping factor rounded to fp32: 6 u of the terms' sizes
  p        the update's relative error is 16 u (moments, corrections, root, division, products) of each of its terms' sizes, the new
           parameter rounds once more: u |p|
  8 bits   the stored code is the lower or the upper neighbour, as y / unit + dither says; fp32 computes y with 16 u, so a code may be
           off by one where y / unit + dither is nearer than that to a whole number
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BLOCK = 64
SIZES = [1, 3, 64, 65, 4095, 4096, 4097, 0, 40001, 255]


def check(name, got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g times the tolerance" % (name, int(bad.sum()), bad.numel(), float(((got.double() - want).abs() / tol).nan_to_num(math.inf).max()))


def make(sizes=SIZES, grad=torch.float32, copy=None, seed=0, shift=0, **kw):
    """An optimizer over views of flat buffers, each starting `shift` elements off its alignment, and its state made up."""
    from wide_deep_amd import optim
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda n, s: torch.randn(n, device="cuda", generator=g) * s
    place = lambda t: torch.cat([t.new_zeros(shift), t])[shift:] if shift else t
    params = [place(rand(n, 0.05)) for n in sizes]
    grads = [place(rand(n, 1e-2).to(grad)) for n in sizes]
    copies = [place(torch.zeros(n, dtype=copy, device="cuda")) for n in sizes] if copy else None
    opt = optim.AdamW(params, grads, lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=[0.1 * (k % 3) for k in range(len(sizes))], copies=copies, **kw)
    m, r = torch.zeros(opt.size, device="cuda"), torch.zeros(opt.size, device="cuda")
    for a, n in zip(opt.starts, sizes):
        m[a: a + n], r[a: a + n] = rand(n, 3e-3), rand(n, 1e-2).abs()
    opt.load_moments(m, r * r if opt.state_bits == 32 else r)
    return opt


def split(opt, flat):
    return [flat[a: a + p.numel()] for a, p in zip(opt.starts, opt.params)]


def decoded(opt):
    """m and v of every tensor in 64 bits, as the state holds them."""
    if opt.state_bits == 32:
        return split(opt, opt.m.double()), split(opt, opt.v.double())
    m, r = opt.moments(torch.float32)
    return split(opt, m.double()), [x * x for x in split(opt, r.double())]


def expected(opt, t, decay):
    """(m, v, p) after step t of each tensor, their tolerances, the global norm."""
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in opt.grads))
    coef = opt.max_norm / max(norm, opt.max_norm) if opt.max_norm else 1.0
    out = []
    for p, g, m, v, d in zip(opt.params, opt.grads, *decoded(opt), decay):
        g, (b1, b2) = g.double() * coef, opt.betas
        tm, tv = 6 * U * (b1 * m.abs() + (1 - b1) * g.abs()), 6 * U * (b2 * v + (1 - b2) * g * g)
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        mh, root = m / (1 - b1 ** t), torch.sqrt(v / (1 - b2 ** t))
        step = opt.lr * (mh / (root + opt.eps) + d * p.double())
        size = opt.lr * ((m.abs() + tm / U / 16) / (1 - b1 ** t) / (root + opt.eps) + d * p.double().abs())
        out.append((m, v, p.double() - step, tm + 1e-45, tv + 1e-45, 16 * U * size + U * p.double().abs() + 1e-45))
    return out, norm


DECAY = [0.1 * (k % 3) for k in range(len(SIZES))]


@pytest.mark.parametrize("grad", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("max_norm,copy,shift", [(None, None, 0), (0.3, torch.bfloat16, 0), (1e3, torch.float16, 1), (0.3, torch.bfloat16, 3)])
def test_steps_with_32_bit_moments(grad, max_norm, copy, shift):
    opt = make(grad=grad, copy=copy, shift=shift, max_norm=max_norm)
    opt.set_step(4)
    for t in (5, 6, 7):
        want, norm = expected(opt, t, DECAY)
        opt.step()
        m, v = decoded(opt)
        for k, (wm, wv, wp, tm, tv, tp) in enumerate(want):
            check("m %d" % k, m[k], wm, tm)
            check("v %d" % k, v[k], wv, tv)
            check("p %d" % k, opt.params[k], wp, tp)
            if copy:
                assert torch.equal(opt.copies[k], opt.params[k].to(copy))
        if max_norm:
            # 16 squares in fp32 (17 roundings at most, of same-signed terms), the rest in 64 bits; the root halves it, one more to store
            assert abs(float(opt.grad_norm) - norm) <= 10 * U * norm
        assert opt.step_count == t
    gap = torch.ones(opt.size, dtype=torch.bool, device="cuda")
    for x in split(opt, gap):
        x.zero_()
    assert bool((opt.m[gap] == 0).all()) and bool((opt.v[gap] == 0).all())


def dither(index, step, seed):
    h = (((index & 0xffffffff) ^ seed) + step * 0x9E3779B1 + (index >> 32) * 0xBB67AE85) & 0xffffffff
    h = ((h ^ (h >> 16)) * 0xBB67AE85) & 0xffffffff
    h = ((h ^ (h >> 15)) * 0x6A09E667) & 0xffffffff
    h = h ^ (h >> 16)
    return (h >> 16).double() / 65536, (h & 0xffff).double() / 65536


def stored(x, d, scale, mantissa, err):
    """What a block of scale byte `scale` stores for x with dither d, and the other neighbour where x is within `err` of a border."""
    unit = torch.exp2(scale.double() - 142.0).repeat_interleave(BLOCK)
    y = x.abs() / unit
    e = torch.floor(torch.log2(y.clamp(min=2.0))).clamp(max=15)
    e = torch.where(torch.exp2(e) > y.clamp(min=2.0), e - 1, e)
    step = torch.exp2(e - mantissa)
    pos = y / step + d
    top = (2.0 - 2.0 ** -mantissa) * 2.0 ** 15
    near = (pos - torch.round(pos)).abs() <= err / unit / step + 2.0 ** -18          # 2^-19 of a step is cut off below the lowest binade
    a = (torch.floor(pos) * step).clamp(max=top)
    b = (torch.where(pos - torch.floor(pos) > 0.5, torch.floor(pos) + 1, torch.floor(pos) - 1).clamp(min=0) * step).clamp(max=top)
    sign = torch.where(x < 0, -1.0, 1.0) * unit
    return a * sign, torch.where(near, b, a) * sign


@pytest.mark.parametrize("grad,copy,shift,max_norm", [(torch.float32, None, 0, None), (torch.bfloat16, torch.bfloat16, 1, 0.2), (torch.float16, torch.float16, 0, 0.2)])
def test_steps_with_8_bit_moments(grad, copy, shift, max_norm):
    opt = make(grad=grad, copy=copy, shift=shift, state_bits=8, seed=3, max_norm=max_norm)
    opt.seed = 77
    opt.set_step(9)
    index = torch.arange(opt.size, device="cuda")
    for t in (10, 11):
        want, _ = expected(opt, t, DECAY)
        opt.step()
        flat = {k: torch.zeros(opt.size, dtype=torch.float64, device="cuda") for k in ("m", "r", "tm", "tr")}
        for k, (wm, wv, wp, tm, tv, tp) in enumerate(want):
            check("p %d" % k, opt.params[k], wp, tp)
            n = slice(opt.starts[k], opt.starts[k] + wm.numel())
            flat["m"][n], flat["r"][n], flat["tm"][n], flat["tr"][n] = wm, wv.sqrt(), tm, 8 * U * wv.sqrt()
            if copy:
                assert torch.equal(opt.copies[k], opt.params[k].to(copy))
        for name, mantissa, d, got, scale in zip("mr", (3, 4), dither(index, t, 77), opt.moments(torch.float32), (opt.m_scale, opt.r_scale)):
            x = flat[name]
            top = x.abs().view(-1, BLOCK).amax(1)
            e = torch.floor(torch.log2(top.clamp(min=2.0 ** -100))) + 127
            sure = (torch.frexp(top.clamp(min=2.0 ** -100))[0] - 0.5 > 1e-6) & (torch.frexp(top.clamp(min=2.0 ** -100))[0] < 1 - 1e-6)
            assert bool((scale.double() == e)[sure].all())
            a, b = stored(x, d, scale, mantissa, flat["t" + name])
            miss = (got.double() != a) & (got.double() != b)
            assert not bool(miss.any()), (name, int(miss.sum()))
            assert float((got.double() != a).double().mean()) < 1e-3


def test_8_bit_values_round_trip_and_bf16_holds_them():
    from wide_deep_amd import optim
    n = 256 * BLOCK
    p = [torch.zeros(n, device="cuda")]
    opt = optim.AdamW(p, [torch.zeros(n, device="cuda")], state_bits=8)
    code = torch.arange(256, device="cuda", dtype=torch.uint8).repeat(BLOCK)
    scale = torch.randint(27, 250, (n // BLOCK,), device="cuda").to(torch.uint8)
    opt.m.copy_(code), opt.r.copy_(code), opt.m_scale.copy_(scale), opt.r_scale.copy_(scale)
    m, r = opt.moments(torch.float32)
    mb, rb = opt.moments()
    assert torch.equal(mb.float(), m) and torch.equal(rb.float(), r)
    c, unit = code.long(), torch.exp2(scale.double() - 142).repeat_interleave(BLOCK)
    value = lambda k, M: torch.where(k >> M == 0, (k & (2 ** M - 1)).double() * 2.0 ** (1 - M), (2.0 ** M + (k & (2 ** M - 1))) * torch.exp2((k >> M).double() - M))
    assert torch.equal(r.double(), value(c, 4) * unit)
    assert torch.equal(m.double(), value(c & 127, 3) * unit * torch.where(c >= 128, -1.0, 1.0))
    # numbers that a block can hold come back as they are
    opt.load_moments(m, r)
    m2, r2 = opt.moments(torch.float32)
    assert torch.equal(m2, m) and torch.equal(r2, r)
    x = torch.randn(n, device="cuda") * torch.exp(3 * torch.randn(n, device="cuda"))
    opt.load_moments(x, x.abs())
    m2, r2 = opt.moments(torch.float32)
    top = x.abs().view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)
    # half a step: 2^-(M + 1) of the binade, above the largest code's value (2 - 2^-M) 2^15 a whole one, and half of the least step below
    check("m", m2, x.double(), 2.0 ** -4 * x.abs().double() + top.double() * 2.0 ** -18)
    check("r", r2, x.abs().double(), 2.0 ** -5 * x.abs().double() + top.double() * 2.0 ** -19)


def test_rounding_is_unbiased_and_slow_moments_move():
    """E[stored] = value: 2^18 copies of one value; the mean's deviation is half a step / 2^9, six of them allowed.  A second moment with
    b2 = 0.999 whose step is a hundredth of a code falls as it should."""
    from wide_deep_amd import optim
    n = 1 << 18
    p, g = [torch.zeros(n, device="cuda")], [torch.zeros(n, device="cuda")]
    opt = optim.AdamW(p, g, state_bits=8, betas=(0.9, 0.999), lr=0.0, weight_decay=0.0)
    m0, r0 = torch.full((n,), 0.0123, device="cuda"), torch.full((n,), 0.0456, device="cuda")
    m0[::BLOCK], r0[::BLOCK] = 0.02, 0.06            # the blocks' largest values
    opt.load_moments(m0, r0)
    m1, r1 = (x.double() for x in opt.moments(torch.float32))
    opt.step()
    m2, r2 = (x.double() for x in opt.moments(torch.float32))
    inner = torch.arange(n, device="cuda") % BLOCK != 0
    for got, want, step in ((m2, m1 * 0.9, 2.0 ** -10), (r2, r1 * math.sqrt(0.999), 2.0 ** -9)):
        assert abs(float((got - want)[inner].mean())) < 6 * step / 2 / 512 + 1e-7
        assert float((got - want)[inner].abs().max()) < step
    for _ in range(99):
        opt.step()
    r3 = opt.moments(torch.float32)[1].double()
    # sqrt is concave by nothing here: a decay is linear in r, so the mean follows exactly; a hundred roundings of half a step at most each
    want = float(r1[inner].mean()) * 0.999 ** 50
    assert abs(float(r3[inner].mean()) - want) < 6 * 10 * 2.0 ** -10 / 512 + 1e-6


def test_step_that_is_not_finite():
    """With clipping it changes nothing and is counted; without, it poisons what it touches: an 8-bit block reads as NaN."""
    for bits in (32, 8):
        opt = make(max_norm=1.0, state_bits=bits)
        opt.step()
        torch.cuda.synchronize()
        was = [x.clone() for x in opt.params + [opt.m, opt.v if bits == 32 else opt.r]]
        for bad in (math.inf, math.nan):
            opt.grads[4][7] = bad
            opt.step()
            assert all(torch.equal(a, b) for a, b in zip(was, opt.params + [opt.m, opt.v if bits == 32 else opt.r]))
        assert opt.skipped == 2 and opt.step_count == 1 and not math.isfinite(float(opt.grad_norm))
        opt.grads[4][7] = 0.5
        opt.step()
        assert opt.step_count == 2 and bool(opt.params[4].isfinite().all())
        opt = make(state_bits=bits)
        opt.grads[4][7] = math.nan
        opt.step()
        assert bool(opt.params[4][7].isnan()) and int(opt.params[4].isnan().sum()) == 1
        if bits == 8:
            m, r = (split(opt, x)[4] for x in opt.moments())
            assert bool(m[:64].isnan().all()) and bool(r[:64].isnan().all()) and bool(m[64:].isfinite().all())


def test_rates_graphs_streams_and_repeats():
    """Two optimizers of one seed give the same bits, eager or replayed; a replay reads the rate from the device and moves the step."""
    from wide_deep_amd import hipgraph
    for bits in (32, 8):
        a, b = (make(max_norm=0.3, state_bits=bits, copy=torch.bfloat16, grad=torch.bfloat16) for _ in range(2))
        rate = torch.tensor([1e-3], device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a.step(lr=rate)
        torch.cuda.synchronize()
        g = hipgraph.new_graph()
        with torch.cuda.graph(g, stream=side):
            a.step(lr=rate)
        b.step(lr=float(rate))
        for k in range(3):
            rate.fill_(1e-3 * (k + 2))
            g.replay()
            torch.cuda.synchronize()
            b.step(lr=float(rate))
            assert all(torch.equal(x, y) for x, y in zip(a.params + a.copies, b.params + b.copies))
            assert torch.equal(a.m, b.m) and a.step_count == b.step_count == k + 2
    with pytest.raises(ValueError, match="lr as a tensor"):
        a.step(lr=torch.tensor([1e-3]))
    with pytest.raises(ValueError, match="state_bits 32"):
        make().moments()
    with pytest.raises(ValueError, match="load_moments"):
        a.load_moments(a.m, a.r)


def test_many_tensors_in_one_step():
    """A thousand tensors of 1 to 2000 elements, more chunks than a launch has workgroups."""
    sizes = [1 + (k * 577) % 2000 for k in range(1000)] + [9000000]
    opt = make(sizes=sizes, max_norm=0.5)
    decay = [0.1 * (k % 3) for k in range(len(sizes))]
    want, norm = expected(opt, 1, decay)
    opt.step()
    assert abs(float(opt.grad_norm) - norm) <= 10 * U * norm
    for k in list(range(0, 1000, 37)) + [1000]:
        check("p %d" % k, opt.params[k], want[k][2], want[k][5])
