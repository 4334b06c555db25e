"""The operators of a training block together: every step of the optimizer, the later ones from moments it holds, against the formula in 64 bits; and samples
whose branches are all dropped."""
import math

import pytest
import torch

from nmrf_amd import optim
from tests.test_training_block import Blocks

pytestmark = pytest.mark.gpu
W, LR, B1, B2, EPS, WD = 2.0 ** -24, 1e-3, 0.9, 0.999, 1e-8, 0.1


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("bits", [32, 8])
def test_every_step_from_the_moments_before_it(kind, bits):
    """m = b1 m + (1 - b1) c g is off by 4 roundings of the first share and 7 of the second, the update by 16 more with sqrt(v)'s, the parameter by 3.  8-bit moments are
    the new ones rounded by less than a code: 2^-4 of the value (sqrt(v): 2^-5) or, below 2^-6 of the scale, 2^-10 (2^-11) of it, a scale being at most twice the
    tensor's largest value."""
    torch.manual_seed(3)
    m = Blocks(96, 200, kind).cuda()
    opt = optim.AdamW([{"params": [p for p in m.parameters() if p.dim() > 1]}, {"params": [p for p in m.parameters() if p.dim() == 1], "weight_decay": 0.0}],
                      lr=LR, weight_decay=WD, state_bits=bits)
    gen = torch.Generator(device="cuda").manual_seed(4)
    held = 0
    for t in range(1, 6):
        x, target = (torch.randn(4, 130, 96, generator=gen, device="cuda") for _ in range(2))
        gates = [(torch.rand(4, 1, 1, generator=gen, device="cuda") < 0.8).float() / 0.8 for _ in range(2)]
        opt.zero_grad()
        ((m(x, gates)[1] - target) ** 2).mean().backward()
        before = {k: (p.detach().double(), p.grad.double(), *((q.double() for q in opt.moments(p)) if t > 1 else (torch.zeros_like(p).double(),) * 2))
                  for k, p in m.named_parameters()}
        opt.step(max_norm=0.05)
        c = min(1.0, 0.05 / (float(opt.grad_norm) + 1e-6))
        for k, p in m.named_parameters():
            p0, g, m0, v0 = before[k]
            a, b = B1 * m0, (1 - B1) * c * g
            m1, v1 = a + b, B2 * v0 + (1 - B2) * (c * g) ** 2
            den = v1.sqrt() / math.sqrt(1 - B2 ** t) + EPS
            want = p0 * (1 - LR * WD * (p.dim() > 1)) - LR / (1 - B1 ** t) * m1 / den
            room = W * (3 * p0.abs() + LR / (1 - B1 ** t) * (4 * a.abs() + 7 * b.abs() + 16 * m1.abs()) / den)
            assert bool(((p.detach().double() - want).abs() <= room).all()), (t, k)
            m2, v2 = (q.double() for q in opt.moments(p))
            if "exp_avg_scale" in opt.state[p]:
                held += t > 1
                r1, r2 = v1.sqrt(), v2.sqrt()
                assert bool(((m2 - m1).abs() <= 2.0 ** -4 * m1.abs() + 2.0 ** -9 * m1.abs().max()).all()), (t, k)
                assert bool(((r2 - r1).abs() <= 2.0 ** -5 * r1 + 2.0 ** -10 * r1.max()).all()), (t, k)
            else:
                assert bool(((m2 - m1).abs() <= W * (4 * a.abs() + 7 * b.abs()) + 1e-44).all()) and bool(((v2 - v1).abs() <= 12 * W * v1 + 1e-44).all()), (t, k)
    assert (held > 0) == (bits == 8)                                # (updates from 8-bit moments were among them)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_samples_whose_branches_are_dropped_pass_through(kind):
    torch.manual_seed(5)
    m = Blocks(96, 200, kind).cuda()
    x = torch.randn(4, 130, 96, device="cuda")
    gates = [torch.tensor(g, device="cuda").view(4, 1, 1) / 0.8 for g in ([0.0, 1.0, 0.0, 1.0], [0.0, 0.0, 1.0, 1.0])]
    out, _ = m(x, gates)
    assert torch.equal(out[0], x[0]) and not any(torch.equal(out[i], x[i]) for i in (1, 2, 3))
