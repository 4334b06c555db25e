"""The gated feed-forward block's activations far from zero (csrc/gated_ffn.hip)."""
import pytest
import torch

from nmrf_amd.ops import gated_ffn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [5, 70])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_far_negative_gates_are_closed(act, dtype, t):
    """One hidden value with u = 1, so that y = act(g): for gelu beyond -7, |g Phi(g)| <= 9e-12 and |slope| <= 6.4e-11 (both largest at -7), for silu
    beyond -30, |g s(g)| <= 2.9e-12 and |slope| <= 2.8e-12.  The forward pass with and without gradients (70 and 5 rows: both of its kernels)."""
    one = torch.ones(1, 1, device="cuda", dtype=dtype)
    for g in (-30.0, -100.0, -1e3, -6e4) + (() if dtype == torch.float16 else (-1e6, -1e20, -1e30)):
        x = torch.full((t, 1), g, device="cuda", dtype=dtype).requires_grad_(True)
        call = lambda: gated_ffn(x, one, one * 0, one, b_up=one[0], act=act)  # noqa: E731
        y = call()
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        with torch.no_grad():
            few = call()
        for v, most in ((y, 1e-11), (few, 1e-11), (dx, 7e-11)):
            assert float(v.detach().double().abs().max()) <= most, (g, float(v.detach().double().abs().max()))
    for g in (30.0, 1e3, 6e4):                                      # and far open ones pass what they get
        x = torch.full((t, 1), g, device="cuda", dtype=dtype).requires_grad_(True)
        y = gated_ffn(x, one, one * 0, one, b_up=one[0], act=act)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert float((y / x.detach() - 1).detach().abs().max()) <= 2.0 ** -20 and float((dx - 1).abs().max()) <= 2.0 ** -20
