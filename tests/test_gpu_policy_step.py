"""GPU: the operators as a program runs them together -- score with the reference policy, loss with the gradient of the logits, AdamW --
on a linear policy logits = x w, eager and as one captured step.  Every step is compared from the same fp32 state with 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class Program:
    """A linear policy of V items over D features, one batch of pairs / sessions, its optimizer."""

    def __init__(self, loss, bits, seed=1):
        from wide_deep_amd import optim
        g = torch.Generator("cuda").manual_seed(seed)
        self.loss, D, V = loss, 24, 1003
        self.lengths = [6, 4, 9, 9, 1, 3]
        T = sum(self.lengths)
        self.x = torch.randn(T, D, device="cuda", generator=g)
        self.w = torch.randn(D, V, device="cuda", generator=g) * 0.2
        self.bias = torch.zeros(V, device="cuda")
        self.w0, self.bias0 = self.w.clone(), self.bias.clone()
        self.targets = torch.randint(0, V, (T,), device="cuda", generator=g, dtype=torch.int32)
        self.targets[:2] = -1
        self.offs = torch.tensor([0] + self.lengths, device="cuda").cumsum(0).to(torch.int32)
        self.adv = torch.randn(len(self.lengths), device="cuda", generator=g)
        self.gw, self.gb = torch.zeros_like(self.w), torch.zeros_like(self.bias)
        self.logits, self.dlogits = torch.empty(T, V, device="cuda"), torch.zeros(T, V, device="cuda")
        self.opt = optim.AdamW([self.w, self.bias], [self.gw, self.gb], lr=1e-2, betas=(0.9, 0.99), weight_decay=[0.1, 0.0], max_norm=0.5, state_bits=bits)
        self.score()

    def forward(self):
        torch.mm(self.x, self.w, out=self.logits)
        self.logits.add_(self.bias)

    def score(self):
        from wide_deep_amd import policy
        self.forward()
        r = policy.sequence_logp(self.logits, self.targets, self.offs)
        self.ref_seq, self.ref_token = r.seq_logp.clone(), r.token_logp.clone()

    def step(self):
        from wide_deep_amd import policy
        self.forward()
        if self.loss == "pair":
            r = policy.preference_loss(self.logits, self.targets, self.offs, ref_logp=self.ref_seq, beta=0.5, reduction="mean", dlogits=self.dlogits)
        else:
            r = policy.policy_loss(self.logits, self.targets, self.offs, self.ref_token, self.adv, ref_logp=self.ref_token, clip=(0.2, 0.2), kl_coef=0.1,
                                   reduction="sequence_mean", dlogits=self.dlogits)
        torch.mm(self.x.t(), self.dlogits, out=self.gw)
        torch.mm(torch.ones(1, len(self.x), device="cuda"), self.dlogits, out=self.gb.view(1, -1))
        self.opt.step()
        return r.loss

    def loss64(self, w, bias):
        """The definition by 64-bit autograd on the CPU."""
        z = self.x.cpu().double() @ w + bias
        t = self.targets.cpu().long()
        lp = torch.where(t >= 0, torch.log_softmax(z, 1).gather(1, t.clamp(min=0).unsqueeze(1)).squeeze(1), 0.0)
        parts = lp.split(self.lengths)
        if self.loss == "pair":
            d = torch.stack([p.sum() for p in parts]) - self.ref_seq.cpu().double()
            return -torch.nn.functional.logsigmoid(0.5 * (d[0::2] - d[1::2])).mean()
        total = 0.0
        for p, old, live, a in zip(parts, self.ref_token.cpu().double().split(self.lengths), (t >= 0).split(self.lengths), self.adv.cpu().double()):
            rho, q = torch.exp(p - old)[live], (old - p)[live]
            total = total + (-torch.minimum(rho * a, rho.clamp(0.8, 1.2) * a) + 0.1 * (torch.exp(q) - q - 1)).mean()
        return total / len(self.lengths)


@pytest.mark.parametrize("loss", ["pair", "policy"])
@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(loss, bits):
    """Gradients against autograd in 64 bits from the same state: products of 24 terms and sums of 32 in fp32, the heads' own roundings
    (about 100 u of the largest, tests of the heads): 256 u of the gradient's norm."""
    a = Program(loss, bits)
    for k in range(6):
        w, bias = (v.cpu().double().requires_grad_() for v in (a.w, a.bias))
        want = a.loss64(w, bias)
        want.backward()
        before = a.w.clone()
        got = a.step()
        assert abs(float(got) - float(want)) < 256 * U * (1 + abs(float(want)))
        for g, v in ((a.gw, w), (a.gb, bias)):
            assert float((g.cpu().double() - v.grad).norm()) < 256 * U * float(v.grad.norm()) + 1e-9
        # the update is bounded by the rate: |m| / root <= 1 / sqrt(1 - b2) with these betas, decay 0.1
        assert 0 < float((a.w - before).abs().max()) < 1e-2 * (10 + 0.1)
    assert a.opt.step_count == 6 and a.opt.skipped == 0


@pytest.mark.parametrize("loss,bits", [("pair", 32), ("policy", 8)])
def test_captured_training_step(loss, bits):
    """One graph holds the whole step; replays are the eager steps bit for bit, with the program's own work in between."""
    from wide_deep_amd import hipgraph
    a, b = Program(loss, bits), Program(loss, bits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.synchronize()
    g = hipgraph.new_graph()
    with torch.cuda.graph(g, stream=side):
        la = a.step()
    b.step()
    for _ in range(4):
        g.replay()
        lb = b.step()
        torch.cuda.synchronize()
        assert torch.equal(la, lb) and torch.equal(a.w, b.w) and torch.equal(a.bias, b.bias) and torch.equal(a.opt.m, b.opt.m)
