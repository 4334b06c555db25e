"""8-bit moments that grow (csrc/adamw.hip): a block's scale doubles where its values stand at the top code and go on growing, so that a moment
that grows by less than a code a step is not held back."""
import math

import pytest
import torch

from nmrf_amd.ops import AdamWPlan, adamw_moment
from tests.test_adamw import _pow2

pytestmark = pytest.mark.gpu
B1, B2, EPS = 0.9, 0.999, 1e-8


def moments(n, dtype=torch.float32):
    z = lambda k, dt: torch.zeros(k, device="cuda", dtype=dt)  # noqa: E731
    blocks = -(-n // 256)
    return z(n, dtype), z(n, torch.uint8), z(n, torch.uint8), z(blocks, torch.float32), z(blocks, torch.float32)


def plan_of(p, m, v, sm, sv):
    return AdamWPlan([p], [m], [v], [sm], [sv])


@pytest.mark.parametrize("grown", [2.2, 2.6])
def test_second_moment_follows_slow_growth(grown):
    """Standard deviation 1.6, then 2.2 or 2.6: sqrt(v) crosses a power of two at 0.01 ... 0.05 % a step.  Bounds of the rounding alone, as for gradients that shrink:
    one code step (<= 2^-5 of the value) is taken with probability d / step, a variance of d * step with d <= 0.0005 times a memory of
    1 / (2 * 0.0005): spread of the logarithm <= sqrt(2^-5 / 2) = 0.125; mean within 0.125^2 of zero (Jensen) plus 0.125 / sqrt(16 384).
    A moment that is cut at every step ends 12 % low.  Looked at every 250 steps from the 750th on (the first ones hold few gradients)."""
    n = 16384
    p, m, v, sm, sv = moments(n)
    plan = plan_of(p, m, v, sm, sv)
    gen = torch.Generator(device="cuda").manual_seed(3)
    vd = torch.zeros(n, device="cuda", dtype=torch.float64)
    for t in range(1, 7001):
        g = torch.randn(n, generator=gen, device="cuda") * (1.6 if t <= 3000 else grown)
        plan.step([g], step=t, lr=1e-4, betas=(B1, B2))
        vd = B2 * vd + (1 - B2) * g.double().square()
        if t >= 750 and t % 250 == 0:
            d = torch.log(adamw_moment(v, sv, squared=True).double().sqrt() / vd.sqrt())
            assert abs(float(d.mean())) <= 0.125 ** 2 + 0.125 / 128 and float(d.std()) <= 0.125, (t, float(d.mean()), float(d.std()))


@pytest.mark.parametrize("level", [1.97, 1.99])
def test_first_moment_reaches_its_level(level):
    """Constant gradients just below a power of two, above the top code 1.9375: rounding is off by at most half a step 2^-4 in standard deviation,
    with a memory of 1 / (1 - 0.9^2): 0.0625 / 2 * 2.3 = 0.072 an element, 0.072 / 128 over 16 384 of them, six times that.  Cut: 1.7 % or more low."""
    n = 16384
    p, m, v, sm, sv = moments(n)
    plan = plan_of(p, m, v, sm, sv)
    g = torch.full((n,), level, device="cuda")
    g[::2] *= -1
    for t in range(1, 301):
        plan.step([g], step=t, lr=1e-4, betas=(B1, B2))
    mean = float((adamw_moment(m, sm).double() * g.sign()).mean())
    assert abs(mean - level * (1 - 0.9 ** 300)) <= 6 * 0.072 / 128, mean


def _codes(a, man, rnd, dropped, scale):
    """Codes of the magnitudes a ([blocks, 256] fp32) under their scales, rounded with the given random bits (in 64 bits, exact)."""
    x = torch.where(scale > 0, a.double() / scale.double().clamp(min=1e-300), torch.zeros_like(a, dtype=torch.float64))
    e = (torch.frexp(x)[1] - 1).clamp(min=-6)
    grid = torch.where(x >= 2.0 ** -6, torch.floor(x * _pow2(23 - e)), torch.floor(x * 2.0 ** 29))
    q = (torch.floor((grid + rnd.double()) / 2.0 ** dropped) * _pow2(e - man)).clamp(max=2 - 2.0 ** -man)
    e = (torch.frexp(q)[1] - 1).clamp(min=-6)
    return torch.where(q >= 2.0 ** -6, (e + 7 << man) + (q * _pow2(-e) - 1) * (1 << man), q * (64 << man)).long()


def _scales(a, old, man):
    top, was = a.amax(-1, keepdim=True), old.amax(-1, keepdim=True)
    s = torch.where(top >= 2.0 ** -100, _pow2(torch.frexp(top)[1] - 1).float(), torch.zeros_like(top))
    edge = s * (2 - 2.0 ** -man)
    return torch.where((top > edge) & (was >= edge), 2 * s, s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_growth_bit_for_bit(dtype):
    """Gradients that grow by 1 % a step (m grows with them, sqrt(v) from 40 % a step down to about 1 %): codes and scales are those of the rule, both where a block's scale doubles
    early and where a value is cut once."""
    n, seed = 256 * 40 + 77, 4
    p, m, v, sm, sv = moments(n, dtype)
    plan = plan_of(p, m, v, sm, sv)
    base = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") * 1e-2
    pad = lambda x: torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)  # noqa: E731
    early = {4: 0, 5: 0}
    cut = {4: 0, 5: 0}
    for t in range(1, 121):
        g = (base * 1.01 ** t).to(dtype)
        mc, vc = adamw_moment(m, sm), adamw_moment(v, sv, squared=True)
        root = adamw_moment(v, sv, squared=True).double().sqrt().float()              # (codes are squares of 6-bit numbers: exact)
        plan.step([g], step=t, lr=1e-3, betas=(B1, B2), seed=seed)
        m1 = mc * torch.tensor(B1, device="cuda") + g.float() * torch.tensor(1 - B1, device="cuda")
        v1 = vc * torch.tensor(B2, device="cuda") + (g.float() * g.float()) * torch.tensor(1 - B2, device="cuda")
        r1 = v1.double().sqrt().float()
        i = torch.arange(n, device="cuda")
        x = (i * 0x9E3779B9 + (seed * 0x9E3779B1 + t * 0xC2B2AE3D & 0xFFFFFFFF)) & 0xFFFFFFFF
        x = ((x ^ (x >> 16)) * 0x6C62272D) & 0xFFFFFFFF
        x = ((x ^ (x >> 15)) * 0x2C9277B5) & 0xFFFFFFFF
        rnd = pad(x ^ (x >> 16))
        for a, old, man, bits, dropped, code, scale in ((m1.abs(), mc.abs(), 4, (rnd >> 18) << 5, 19, m.long() & 127, sm),
                                                        (r1, root, 5, rnd & 0x3FFFF, 18, v.long(), sv)):
            s = _scales(pad(a), pad(old), man)
            want = _codes(pad(a), man, bits, dropped, s)
            if man == 5:
                want = torch.where((pad(a) > 0) & (s > 0), want.clamp(min=1), want)
            assert torch.equal(scale, s.squeeze(1)) and torch.equal(code, want.view(-1)[:n]), (t, man)
            top = pad(a).amax(-1)
            early[man] += int((scale > top).sum())
            cut[man] += int(((scale <= top) & (top > scale * (2 - 2.0 ** -man))).sum())
        assert torch.equal(m.long() >> 7 & (m.long() & 127 > 0), (m1 < 0).long() & (m.long() & 127 > 0))
    assert min(early.values()) > 0 and min(cut.values()) > 0, (early, cut)


def test_scale_at_the_end_of_the_range():
    """2^127 cannot double: the largest finite first moments keep the top code."""
    p, m, v, sm, sv = moments(256)
    m[:], sm[:] = 127, 2.0 ** 127
    plan_of(p, m, v, sm, sv).step([torch.full((256,), 3.4e38, device="cuda")], step=1, lr=0.0, betas=(B1, B2))
    assert float(sm[0]) == 2.0 ** 127 and bool((m == 127).all()) and math.isnan(float(sv[0]))
