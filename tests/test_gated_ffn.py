"""The gated feed-forward block (csrc/gated_ffn.hip, nmrf_amd.ops.gated_ffn) against the formula in 64 bits, its gradients against autograd of
that formula and against differences of the kernel's own forward pass.

Tolerances, for an output that is a sum of n products a_i b_i in fp32 (the matrix pipe adds in some order: at most n roundings, in practice a
few): |error| <= (sqrt(n) + 16) 2^-24 sum |a_i b_i|, with the elements' own errors on top: in 16-bit types every intermediate that is stored
(h, g, u, dg, du) is off by half a step u of its value, which passes into the sum as u sum |a_i b_i| / sqrt(n) for roundings of random sign;
fp32 operands are fp16 pairs, 2^-22 of the value and 2^-38 of the tensor's largest entry.  The sums of magnitudes are formed in 64 bits beside
the result.  A factor of 6 for the largest of up to 10^6 elements (normal deviates)."""
import math

import pytest
import torch

from nmrf_amd import _lib
from nmrf_amd.ops import gated_ffn

W = 2.0 ** -24
U = {torch.float32: 2.0 ** -22, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NAMES = ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")


def act_and_slope(g, act):
    if act == "relu":
        return torch.relu(g), (g > 0).to(g.dtype)
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    phi = torch.special.ndtr(g)
    return g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def case(t, d, f, do, dtype, bias, seed=0, odd=False, lead=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, std=1.0):
        n = math.prod(shape)
        flat = torch.empty(n + 8, device="cuda", dtype=dtype)
        return flat[1 if odd else 0:][:n].view(shape).copy_(torch.randn(shape, generator=gen, device="cuda") * std)
    v = {"x": rand(*(lead or (t,)), d), "w_gate": rand(f, d, std=d ** -0.5), "w_up": rand(f, d, std=d ** -0.5), "w_down": rand(do, f, std=f ** -0.5),
         "b_gate": rand(f, std=0.2) if bias else None, "b_up": rand(f, std=0.2) if bias else None, "b_down": rand(do, std=0.2) if bias else None}
    return v, rand(*(lead or (t,)), do, std=0.3)


def formula(v, dy, act):
    """Values, gradients and for each the sum of the magnitudes behind it, in 64 bits."""
    r = {k: None if x is None else x.detach().double().reshape(-1, x.shape[-1]) if k == "x" else x.detach().double() for k, x in v.items()}
    dy = dy.double().reshape(-1, dy.shape[-1])
    a = {k: None if x is None else x.abs() for k, x in r.items()}
    b = lambda z, q: z if q is None else z + q  # noqa: E731
    g, u = b(r["x"] @ r["w_gate"].t(), r["b_gate"]), b(r["x"] @ r["w_up"].t(), r["b_up"])
    mg, mu = b(a["x"] @ a["w_gate"].t(), a["b_gate"]), b(a["x"] @ a["w_up"].t(), a["b_up"])
    ac, sl = act_and_slope(g, act)
    h = ac * u
    # what an error of g and u (as large as their magnitude sums, relatively) makes of h, dg, du: |act'| <= 1.13, |act''| <= 0.8
    mh = ac.abs() * mu + 1.13 * mg * u.abs()
    dh = dy @ r["w_down"]
    mdh = dy.abs() @ a["w_down"]
    du, dg = dh * ac, dh * u * sl
    mdu, mdg = mdh * ac.abs() + dh.abs() * 1.13 * mg, mdh * u.abs() * 1.13 + dh.abs() * (mu * 1.13 + u.abs() * 0.8 * mg)
    out = {"y": (b(h @ r["w_down"].t(), r["b_down"]), b(mh @ a["w_down"].t(), a["b_down"])),
           "x": (dg @ r["w_gate"] + du @ r["w_up"], mdg @ a["w_gate"] + mdu @ a["w_up"]),
           "w_gate": (dg.t() @ r["x"], mdg.t() @ a["x"]), "w_up": (du.t() @ r["x"], mdu.t() @ a["x"]), "w_down": (dy.t() @ h, dy.abs().t() @ mh),
           "b_gate": (dg.sum(0), mdg.sum(0)), "b_up": (du.sum(0), mdu.sum(0)), "b_down": (dy.sum(0), dy.abs().sum(0))}
    d, f, do, t = r["x"].shape[1], r["w_gate"].shape[0], dy.shape[1], dy.shape[0]
    n = {"y": f + d, "x": 2 * f + do, "w_gate": t + do, "w_up": t + do, "w_down": t + d, "b_gate": t + do, "b_up": t + do, "b_down": t}
    return out, n


def run(v, dy, act, grad=True):
    leaves = {k: None if t is None else t.detach().requires_grad_(grad) for k, t in v.items()}
    y = gated_ffn(*[leaves[k] for k in NAMES], act=act)
    if not grad:
        return y, None
    names = [k for k in NAMES if leaves[k] is not None]
    return y, dict(zip(names, torch.autograd.grad(y, [leaves[k] for k in names], dy)))


def check(v, dy, act, grad=True):
    y, grads = run(v, dy, act, grad)
    want, n = formula(v, dy, act)
    dtype = v["x"].dtype
    got = {"y": y, **(grads or {})}
    for k, a in got.items():
        ref, mag = want[k]
        assert a.dtype == dtype and a.shape == (v[k].shape if k in v else (*v["x"].shape[:-1], dy.shape[-1])), k
        a = a.double().reshape(ref.shape)
        store = U[dtype] if dtype != torch.float32 else 0.0
        tol = store * ref.abs() + 6 * mag * ((math.sqrt(n[k]) + 16) * W + 2 * U[dtype] / math.sqrt(n[k])) + 64 * 2.0 ** -38 * mag.max()
        if dtype == torch.float16:                                  # h, dg, du below 2^-14 lose bits: half of 2^-24 each, times the other factor
            tol = tol + 2.0 ** -24 + 6 * 2.0 ** -25 * math.sqrt(n[k]) * (1 if k not in v else 1)
        bad = (a - ref).abs() > tol
        assert not bool(bad.any()), (k, tuple(a.shape), float(((a - ref).abs() / tol).max()), int(bad.sum()))
    return y, grads


# ---- refusals: on the host ------------------------------------------------------------------------------------------------------------
def test_refusals():
    x, w, wd = torch.zeros(3, 8), torch.zeros(16, 8), torch.zeros(8, 16)
    with pytest.raises(_lib.NmrfHipError, match="MI355X only"):
        gated_ffn(x, w, w, wd)
    with pytest.raises(ValueError, match="act"):
        gated_ffn(x, w, w, wd, act="tanh")
    for args, what in (((x, w, w[:8], wd), "w_up"), ((x, w, w, wd[:, :8]), "w_down"), ((x, w[:, :4], w, wd), "w_gate"), ((x, w[0], w, wd), "x"),
                       ((x, w, w, wd, torch.zeros(8)), "b_gate"), ((x, w, w, wd, None, None, torch.zeros(16)), "b_down"),
                       ((x[:, :0], w[:, :0], w[:, :0], wd), "widths")):
        with pytest.raises(ValueError, match=what):
            gated_ffn(*args)


def test_c_entries_refuse_before_they_launch():
    lib = _lib.load()

    def fwd(x=64, t=4, d=8, f=8, do=8, dtype=1, act=0, h=64, g=None, u=None, y=64, amax=None, ws=64, floats=1 << 30):
        return lib.nmrf_gated_ffn(x, 64, 64, 64, None, None, None, t, d, f, do, dtype, act, h, g, u, y, amax, ws, floats, None)
    assert fwd(t=0) == 0
    assert fwd(x=None) == -3 and fwd(h=None) == -3 and fwd(y=None) == -3 and fwd(dtype=0) == -3
    for bad in (dict(t=-1), dict(d=0), dict(f=0), dict(do=0), dict(d=(1 << 22) + 1), dict(dtype=3), dict(act=3), dict(g=64), dict(x=65), dict(y=65),
                dict(x=66, dtype=0, amax=64), dict(dtype=0, amax=66), dict(t=0x7fffffff), dict(g=66, u=64), dict(ws=66), dict(t=200, f=8192, floats=0)):
        assert fwd(**bad) == -1, bad

    def bwd(t=4, dtype=1, ws=64, floats=1 << 30, dg=64, amax=None):
        return lib.nmrf_gated_ffn_bwd(64, 64, 64, 64, 64, 64, 64, 64, t, 8, 8, 8, dtype, 0, dg, 64, 64, None, None, None, None, None, None, amax, ws, floats, None)
    assert bwd(t=0) == -1 and bwd(ws=None) == -3 and bwd(dg=None) == -3 and bwd(dtype=0) == -3 and bwd(floats=0) == -1 and bwd(ws=66) == -1 and bwd(dg=65) == -1
    import ctypes
    n = ctypes.c_int64()
    size = lambda t, back, p=ctypes.byref(n): lib.nmrf_gated_ffn_size(t, 128, 512, 128, 0, back, p)  # noqa: E731
    assert size(-1, 1) == -1 and size(4, 1, None) == -3 and size(0, 1) == 0 and n.value == 0
    assert size(29952, 1) == 0 and n.value > 2 * 128 * 512 and size(29952, 0) == 0 and n.value == 0


# ---- the formula ------------------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1, 1), (1, 8, 8, 8), (3, 17, 33, 5), (16, 64, 128, 64), (17, 40, 72, 24), (64, 96, 200, 96), (65, 128, 64, 128), (127, 33, 129, 65),
          (128, 128, 128, 128), (129, 136, 264, 72), (300, 321, 861, 321), (777, 64, 100, 48), (1000, 128, 512, 128), (5000, 72, 136, 40),
          (200, 1, 3, 2), (321, 3, 1, 7), (2100, 200, 130, 9), (450, 700, 1030, 60)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, dtype):
    i = SHAPES.index(shape)
    v, dy = case(*shape, dtype, bias=i % 2 == 0, seed=i, odd=i % 3 == 2)
    act = ("silu", "gelu", "relu")[i % 3]
    if act == "relu":                                               # the slope jumps at zero: keep g away from it by more than its error
        v["b_gate"] = torch.full((shape[2],), 0.05, device="cuda", dtype=dtype)
        g = v["x"].double() @ v["w_gate"].double().t() + v["b_gate"].double()
        v["x"][g.abs().min(1).values < 1e-2] = 0.0
    check(v, dy, act)
    check(v, dy, act, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 32, 33, 48, 49, 64])
def test_few_tokens(t, dtype):
    v, dy = case(t, 520, 1000 + t, 257, dtype, bias=t % 2 == 0, seed=t, odd=t % 3 == 0)
    check(v, dy, "silu", grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_tiles(dtype):
    """Enough tiles of 256 x 256 to be chosen, none of them whole at the edges; weight gradients with and without a split contraction."""
    v, dy = case(4099, 520, 1600, 515, dtype, True, seed=21)
    check(v, dy, "silu")


@pytest.mark.gpu
def test_no_gradient_mode_takes_the_short_way():
    """Parameters that require gradients under no_grad: the same call as without them, bit for bit (one token: the weights are streamed)."""
    for t in (1, 200):
        v, dy = case(t, 64, 96, 48, torch.bfloat16, True, seed=22)
        want, _ = run(v, dy, "silu", grad=False)
        leaves = {k: x.clone().requires_grad_(True) for k, x in v.items()}
        with torch.no_grad():
            y = gated_ffn(*[leaves[k] for k in NAMES])
        assert torch.equal(y, want) and not y.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_leading_dimensions_and_shared_rows(act):
    v, dy = case(0, 64, 96, 80, torch.float32, True, seed=3, lead=(2, 3, 35))
    if act == "relu":
        v["b_gate"] = torch.full((96,), 3.0, device="cuda")         # (far from the jump)
        v["x"] *= 0.2
    y, grads = check(v, dy, act)
    x = v["x"].transpose(0, 2)                                       # other strides, same values
    again = gated_ffn(x, *[v[k] for k in NAMES[1:]], act=act)
    assert torch.equal(again.transpose(0, 2), y)
    one = v["x"][:1, :1, :1].expand(2, 3, 35, 64)                    # a broadcast input: its gradient is summed by autograd
    leaf = one[:1, :1, :1].clone().requires_grad_(True)
    gated_ffn(leaf.expand(2, 3, 35, 64), *[v[k] for k in NAMES[1:]], act=act).backward(dy)
    full = one.clone().requires_grad_(True)
    gated_ffn(full, *[v[k] for k in NAMES[1:]], act=act).backward(dy)
    s = full.grad.double().sum((0, 1, 2))
    assert float((leaf.grad.double().view(-1) - s).abs().max()) <= 210 * W * float(full.grad.abs().sum((0, 1, 2)).max())


@pytest.mark.gpu
def test_fp32_operands_of_very_different_size():
    """The power-of-two scaling: gradients of a mean loss and weights near the fp16 limit keep their bits."""
    v, dy = case(300, 64, 96, 64, torch.float32, False, seed=4)
    for a, b, c in ((1e-6, 1.0, 1e-7), (3e4, 1e-4, 1e-12), (1.0, 1e5, 1e-3)):
        w = {**v, "x": v["x"] * a, "w_gate": v["w_gate"] / a, "w_up": v["w_up"] * b, "w_down": v["w_down"] / b}
        check(w, dy * c, "silu")
    z = {k: None if t is None else torch.zeros_like(t) for k, t in v.items()}
    y, grads = run(z, dy, "gelu")
    assert not bool(y.any()) and not any(bool(g.any()) for g in grads.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_that_are_not_finite_stay_in_their_row(dtype):
    v, dy = case(200, 64, 96, 48, dtype, False, seed=5)
    v["x"][7, 3], v["x"][150, 0] = float("nan"), float("inf")
    y, _ = run(v, dy, "silu", grad=False)
    keep = torch.ones(200, dtype=torch.bool, device="cuda")
    keep[[7, 150]] = False
    assert bool(torch.isfinite(y[keep]).all()) and bool(torch.isnan(y[7]).all()) and not bool(torch.isfinite(y[150]).any())
    if dtype == torch.float32:                                      # a row that is not finite leaves the scale to the others, large or small
        for c in (1e7, 1e-7):
            w = {**v, "x": v["x"] * c, "w_gate": v["w_gate"] / c, "w_up": v["w_up"] / c}
            other, _ = run(w, dy, "silu", grad=False)
            want, _ = formula({**w, "x": torch.where(keep[:, None], w["x"], torch.zeros_like(w["x"]))}, dy, "silu")
            assert float((other[keep].double() - want["y"][0][keep]).abs().max()) <= 6 * (math.sqrt(160) + 16 + 8) * W * float(want["y"][1].max())
    few, _ = run({**v, "x": v["x"][:20]}, dy[:20], "silu", grad=False)
    assert bool(torch.isnan(few[7]).all()) and bool(torch.isfinite(few[[i for i in range(20) if i != 7]]).all())


@pytest.mark.gpu
def test_gradients_against_differences_of_the_forward_pass():
    """Central differences of the kernel in fp32 at steps e and 2 e, extrapolated (off by O(e^4)); L = <A, y> is summed in 64 bits from outputs whose
    errors (64 * 2^-24 of O(1) values, N of them, random signs) are divided by e = 2^-5."""
    v, a = case(70, 40, 56, 24, torch.float32, True, seed=6)
    _, grads = run(v, a, "silu")
    gen = torch.Generator(device="cuda").manual_seed(7)
    loss = lambda w: float((run(w, None, "silu", grad=False)[0].double() * a.double()).sum())  # noqa: E731
    for k in NAMES:
        d = torch.randn(v[k].shape, generator=gen, device="cuda")
        d = d / d.norm() * 2
        e = 2.0 ** -5
        dd = [(loss({**v, k: v[k] + s * e * d}) - loss({**v, k: v[k] - s * e * d})) / (2 * s * e) for s in (1, 2)]
        got = float((grads[k].double() * d.double()).sum())
        assert abs((4 * dd[0] - dd[1]) / 3 - got) <= 64 * W * math.sqrt(a.numel()) * 0.3 * 2 / e + 1e-3 * abs(got) + 1e-4, (k, dd, got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_only_what_is_asked_for(dtype):
    v, dy = case(200, 64, 96, 48, dtype, True, seed=8)
    _, full = run(v, dy, "gelu")
    for some in (("x",), ("w_gate",), ("w_up", "b_down"), ("w_down", "b_gate", "x")):
        leaves = {k: v[k].detach().requires_grad_(k in some) for k in NAMES}
        y = gated_ffn(*[leaves[k] for k in NAMES], act="gelu")
        for k, g in zip(some, torch.autograd.grad(y, [leaves[k] for k in some], dy)):
            assert torch.equal(g, full[k]), (k, some)


@pytest.mark.gpu
def test_repeats_streams_and_second_backward():
    v, dy = case(900, 128, 192, 128, torch.float32, True, seed=9)
    one = run(v, dy, "silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        two = run(v, dy, "silu")
    torch.cuda.current_stream().wait_stream(s)
    leaves = {k: v[k].detach().requires_grad_(True) for k in NAMES}
    y = gated_ffn(*[leaves[k] for k in NAMES], act="silu")
    first = torch.autograd.grad(y, list(leaves.values()), dy * 1e-6, retain_graph=True)
    again = torch.autograd.grad(y, list(leaves.values()), dy)
    for k, g in zip(NAMES, again):
        assert torch.equal(g, one[1][k]) and torch.equal(g, two[1][k]), k
    assert torch.equal(one[0], two[0]) and torch.equal(one[0], y) and bool(torch.isfinite(first[0]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("t,dtype", [(1, torch.bfloat16), (200, torch.bfloat16), (200, torch.float32)])
def test_forward_is_captured_and_backward_refuses(t, dtype):
    v, dy = case(t, 64, 96, 64, dtype, True, seed=10)
    call = lambda: gated_ffn(*[v[k] for k in NAMES])  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for _ in range(3):
        v["x"].mul_(-0.75)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    x = v["x"].clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(_lib.NmrfHipError, match="not captured"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(gated_ffn(x, *[v[k] for k in NAMES[1:]]), x, dy)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_no_rows_and_refusals_on_the_device():
    v, dy = case(0, 16, 24, 8, torch.bfloat16, True, seed=11)
    y, grads = run(v, dy, "silu")
    assert y.shape == (0, 8) and not any(bool(g.any()) for g in grads.values())
    v, _ = case(4, 16, 24, 8, torch.float32, False, seed=11)
    with pytest.raises(_lib.NmrfHipError, match="expected"):
        gated_ffn(v["x"], v["w_gate"].bfloat16(), v["w_up"], v["w_down"])
    with pytest.raises(_lib.NmrfHipError, match="fp32, bf16 or fp16"):
        gated_ffn(v["x"].double(), v["w_gate"].double(), v["w_up"].double(), v["w_down"].double())
