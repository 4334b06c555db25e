"""The summed gradients of residual_norm -- parameters and shared gates -- against the formula in 64 bits, each within (400 + sqrt(terms)) 2^-24 of the sum of its
terms' magnitudes (formed in 64 bits beside the reference: at every subtraction the magnitudes are added), and that bound within 3 % of the
largest value it is a bound for: a gradient of zero or of the other sign does not pass."""
import math

import pytest
import torch

from tests.test_residual_norm import NAMES, formula, run

W = 2.0 ** -24


def inputs(shape, gate, device):
    """Made on the CPU, so that the reference alone can be looked at there.  The outputs' gradients lean on y: the sums do not cancel."""
    gen = torch.Generator().manual_seed(17)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    c = shape[-1]
    y = r(*shape) - 0.3
    v = {"x": 2 * r(*shape) + 0.5, "y": y, "gate": 0.7 * r(*gate) + 0.2, "scale": torch.rand(c, generator=gen) + 0.5,
         "post_w": torch.rand(c, generator=gen) + 0.5, "post_b": 0.3 * r(c), "next_w": torch.rand(c, generator=gen) + 0.5, "next_b": 0.3 * r(c)}
    d_out, d_h = 0.3 * r(*shape) + 0.2 * y + 0.1, 0.3 * r(*shape) + 0.1 * y + 0.1
    return {k: t.to(device) for k, t in v.items()}, d_out.to(device), d_h.to(device)


def reference(v, d_out, d_h, kind, act):
    """-> {name: (gradient, room)}, room: 2^-24 (400 + sqrt(terms)) sum |terms|"""
    q = {k: t.detach().double().requires_grad_(True) for k, t in v.items()}
    if kind == "rms":
        q["post_b"] = q["next_b"] = None
    outs = formula(q, kind, True, True, act, 1.0, 1e-5)
    names = [k for k in NAMES if q[k] is not None]
    grads = dict(zip(names, torch.autograd.grad(outs, [q[k] for k in names], (d_out.double(), d_h.double()))))
    q = {k: None if t is None else t.detach() for k, t in q.items()}

    def norm(z):                                                    # (normalised values, magnitudes behind them, 1 / deviation)
        mean = z.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(z[..., :1])
        rs = 1 / torch.sqrt(((z - mean) ** 2).mean(-1, keepdim=True) + 1e-5)
        return (z - mean) * rs, (z.abs() + mean.abs()) * rs, rs
    _, mz, _ = norm(q["y"])
    g = q["gate"]
    a, slope = {None: (g, torch.ones_like(g)), "sigmoid": (torch.sigmoid(g), torch.sigmoid(g) * (1 + torch.sigmoid(g))), "tanh": (torch.tanh(g), 1 + torch.tanh(g) ** 2)}[act]
    _, mh, hr = norm(outs[0].detach())
    hh = norm(outs[0].detach())[0]
    u = (d_h.double() * q["next_w"]).abs()
    mdx = d_out.double().abs() + hr * (u + (u.mean(-1, keepdim=True) if kind == "layer" else 0) + hh.abs() * (u * hh.abs()).mean(-1, keepdim=True))
    full = mz * q["post_w"] + (0 if q["post_b"] is None else q["post_b"].abs())
    terms = {"gate": mdx * full * q["scale"] * slope, "scale": mdx * full * a.abs(), "post_w": mdx * (q["scale"] * a).abs() * mz, "post_b": mdx * (q["scale"] * a).abs(),
             "next_w": d_h.double().abs() * mh, "next_b": d_h.double().abs()}
    out = {}
    for k, m in terms.items():
        if q[k] is not None:
            to = q[k].shape
            n = m.numel() // q[k].numel()
            out[k] = grads[k], W * (400 + math.sqrt(n)) * m.sum_to_size((1,) * (m.dim() - len(to)) + tuple(to)).view(to)
    return out


CASES = [((2, 300, 256), g) for g in ((2, 300, 1), (2, 1, 256), (2, 1, 1), (256,), (1,))] + [
    ((5, 41, 72), (5, 1, 72)), ((5, 41, 72), (1,)), ((3, 2, 7, 48), (3, 1, 1, 48)), ((3, 2, 7, 48), (3, 2, 1, 1)), ((2, 2500, 64), (2, 1, 1)),
    ((2, 2500, 64), (64,)), ((2, 700, 600), (2, 1, 1)), ((1, 900, 2500), (2500,)), ((3, 50, 4100), (3, 1, 1)), ((700, 3, 32), (700, 1, 1))]


def judged(v, d_out, d_h, kind, act):
    want = reference(v, d_out, d_h, kind, act)
    for k, (ref, room) in want.items():
        assert float(room.max()) <= 0.03 * float(ref.abs().max()), (k, float(room.max()), float(ref.abs().max()))
    return want


@pytest.mark.parametrize("shape,gate", [c for c in CASES if math.prod(c[0]) <= 160000])
def test_bounds_are_small_beside_what_they_bound(shape, gate):
    for kind, act in (("layer", None), ("rms", "sigmoid"), ("layer", "tanh")):
        judged(*inputs(shape, gate, "cpu"), kind, act)


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "sigmoid", "tanh"])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("shape,gate", CASES)
def test_summed_gradients(shape, gate, kind, act):
    v, d_out, d_h = inputs(shape, gate, "cuda")
    want = judged(v, d_out, d_h, kind, act)
    if kind == "rms":
        v["post_b"] = v["next_b"] = None
    _, grads = run(v, d_out, d_h, kind, act)
    for k, (ref, room) in want.items():
        bad = (grads[k].double() - ref).abs() > room
        assert not bool(bad.any()), (k, float(((grads[k].double() - ref).abs() / room).max()))
