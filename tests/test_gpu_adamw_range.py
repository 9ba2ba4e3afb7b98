"""GPU: AdamW at the ends of its ranges (csrc/adamw.hip) -- blocks whose elements differ by many powers of two, limits of the norm; u = 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BLOCK = 64


@pytest.mark.parametrize("ratio", [1e2, 1e4, 1e5, 1e6, 1e7])
@pytest.mark.parametrize("b2", [0.95, 0.999])
@pytest.mark.parametrize("kind", ["steady", "spike"])
def test_small_elements_beside_a_large_one(ratio, b2, kind):
    """8-bit moments, one element of each block with gradients `ratio` times its neighbours', always or once.  A neighbour's root may be stored
    as code 0 under a first moment that is not 0: the step reads code 0 as code 1, so that no update is of the size m / eps.

    Each step is checked against the formula on the state as it stands (tolerance: 16 u of the update's terms, as everywhere for AdamW), and no
    neighbour moves by more than 32 lr.  That bound: in 32 bits |m| <= K sqrt(v), K = (1 - b1) / sqrt((1 - b2)(1 - b1^2 / b2)) <= 7.3, so the
    scale bytes are at most 3 apart; code 1 of m is then at most 2^(3 + 1) times code 1 of r, and twice that is allowed for roundings that
    went up; the corrections' ratio is at most 2.24 where K is 1.2 (b2 0.95) and at most 1 where it is 7.3."""
    from wide_deep_amd import optim
    n, b1, lr, eps = 256 * BLOCK, 0.9, 1.0, 1e-8
    gen = torch.Generator("cuda").manual_seed(int(ratio) % 1000 + 5)
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    opt = optim.AdamW([p], [g], lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0, state_bits=8)
    large = torch.arange(n, device="cuda") % BLOCK == 0
    zeros = 0
    for t in range(1, 61):
        g.copy_(torch.randn(n, device="cuda", generator=gen) * 1e-3)
        if kind == "steady" or t == 10:
            g[large] *= ratio
        m, r = (x.double() for x in opt.moments(torch.float32))
        zeros += int(((r == 0) & (m != 0)).sum())
        least = torch.exp2(opt.r_scale.double() - 145.0).repeat_interleave(BLOCK)          # code 1
        old = p.double()
        opt.step()
        g64 = g.double()
        m, v = b1 * m + (1 - b1) * g64, b2 * torch.maximum(r, least) ** 2 + (1 - b2) * g64 * g64
        size = lr / (1 - b1 ** t) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
        tol = 16 * U * size * (m.abs() + 6 / 16 * ((m - (1 - b1) * g64).abs() + (1 - b1) * g64.abs())) + U * old.abs() + 1e-45
        off = (p.double() - (old - size * m)).abs() / tol
        assert float(off.max()) <= 1.0, (t, float(off.max()))
        assert float((p.double() - old)[~large].abs().max()) <= 32 * lr, t
    assert zeros > 0 or ratio < 1e5 or (kind == "spike" and ratio < 1e6)                   # the cases that matter were met


def test_loaded_roots_of_code_zero():
    """Numbers of a checkpoint far below their block's largest root: loaded to nearest they are code 0, and the next step stays bounded."""
    from wide_deep_amd import optim
    n = 4 * BLOCK
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    opt = optim.AdamW([p], [g], lr=1.0, weight_decay=0.0, state_bits=8)
    m, r = torch.full((n,), 1e-3, device="cuda"), torch.full((n,), 1e-3, device="cuda")
    r[::BLOCK] = 1e4
    opt.load_moments(m, r)
    opt.set_step(1000)
    assert int((opt.r == 0).sum()) == n - n // BLOCK
    opt.step()
    # code 1 is 2^-18 of 2^13 <= 1e4: the update is 0.9e-3 / (2^-5 sqrt(0.999) / sqrt(1 - 0.999^1001)) = 0.023
    want = 0.9e-3 / (2.0 ** -5 * math.sqrt(0.999 / (1 - 0.999 ** 1001)))
    # m was rounded to a code: half a step of 3 bits
    assert abs(float(p[1]) + want) <= want / 16 + 1e-6 and bool((p.abs() <= 0.03).all())
    # a block that holds nothing but zeros still holds nothing
    opt.load_moments(torch.zeros_like(m), torch.zeros_like(r))
    p.zero_()
    opt.step()
    assert bool((p == 0).all()) and bool((opt.r == 0).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_an_infinite_max_norm_only_tells_the_norm(bits):
    from wide_deep_amd import optim
    sizes = [5, 64, 4099]

    def run(max_norm):
        gen = torch.Generator("cuda").manual_seed(3)
        p = [torch.randn(n, device="cuda", generator=gen) for n in sizes]
        g = [torch.randn(n, device="cuda", generator=gen) for n in sizes]
        opt = optim.AdamW(p, g, max_norm=max_norm, state_bits=bits)
        for _ in range(3):
            opt.step()
        return opt

    a, b = run(None), run(math.inf)
    assert all(torch.equal(x, y) for x, y in zip(a.params + [a.m], b.params + [b.m])) and all(bool(x.isfinite().all()) for x in b.params)
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in b.grads))
    assert abs(float(b.grad_norm) - norm) <= 10 * U * norm and b.step_count == 3 and b.skipped == 0
    b.grads[1][3] = math.inf
    b.step()
    assert b.skipped == 1 and all(torch.equal(x, y) for x, y in zip(a.params, b.params))


def test_a_max_norm_that_is_no_fp32_number_is_refused():
    """2^-150 reaches the kernel as 0, which means no clipping."""
    from wide_deep_amd import optim
    p, g = [torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda")]
    for bad in (0.0, -1.0, 2.0 ** -151, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            optim.AdamW(p, g, max_norm=bad)
    optim.AdamW(p, g, max_norm=2.0 ** -149).step()


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
def test_largest_gradients_of_a_clipped_step(grad):
    """The squares of eight elements are added in fp32: sqrt(2^128 / 8) = 6.5e18 is what all of them may be."""
    from wide_deep_amd import optim
    n = 4 * 2048 + 77
    p = torch.zeros(n, device="cuda")
    g = torch.full((n,), 6.4e18, device="cuda").to(grad)
    opt = optim.AdamW([p], [g], lr=1.0, max_norm=1.0, weight_decay=0.0)
    opt.step()
    norm = math.sqrt(n) * float(g[0].double())
    assert opt.skipped == 0 and opt.step_count == 1 and abs(float(opt.grad_norm) - norm) <= 10 * U * norm
    # first step, all alike: m / sqrt(v) of the corrected moments is 1 (g' = n^-1/2 is far above eps)
    assert bool(((p + 1.0).abs() <= 1e-5).all())
    was = p.clone()
    g.fill_(7e18)
    opt.step()
    assert opt.skipped == 1 and opt.step_count == 1 and torch.equal(p, was)


def test_one_gradient_whose_square_is_not_finite():
    """With clipping the step is skipped; without, 32 bits keep the parameter where it is (m / inf); 8 bits square after
    the product with 1 - b2, 0.001 (2e19)^2 = 4e35 is in range, and keep the root."""
    from wide_deep_amd import optim
    for bits in (32, 8):
        p, g = torch.zeros(256, device="cuda"), torch.full((256,), 1e-3, device="cuda")
        g[70] = 2e19
        opt = optim.AdamW([p], [g], lr=1.0, max_norm=1.0, weight_decay=0.0, state_bits=bits)
        opt.step()
        assert opt.skipped == 1 and bool((p == 0).all())
        opt = optim.AdamW([p], [g], lr=1.0, weight_decay=0.0, state_bits=bits)
        opt.step()
        others = torch.arange(256, device="cuda") != 70
        assert bool(((p[others] + 1).abs() < 1e-3).all())
        if bits == 32:
            assert float(p[70]) == 0.0 and float(opt.v[70]) == math.inf
        else:
            m, r = opt.moments(torch.float32)
            assert abs(float(p[70]) + 1) < 1e-3 and bool(m.isfinite().all()) and bool(r.isfinite().all())
            assert abs(float(r[70]) / (math.sqrt(0.001) * 2e19) - 1) <= 2.0 ** -4         # a step of 4 bits
            g[70] = 1e21                                                                  # 0.001 (1e21)^2 = 1e39 is not
            opt.step()
            m, r = opt.moments()
            assert bool(p[70].isnan()) and bool(r[64:128].isnan().all()) and bool(r[:64].isfinite().all()) and bool(r[128:].isfinite().all())
