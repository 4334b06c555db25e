"""The norms around a block with its gate and residual scale (csrc/residual_norm.hip, nmrf_amd.ops.residual_norm) against the formula in 64
bits, its gradients against autograd of that formula and against differences of the kernel's own forward pass.

Tolerances: an output is rounded once to its type (half a step, u |value|).  Before that, a row goes through at most two norms (16 additions in a
lane and 9 levels between lanes for each statistic), one backward dot of the same length for each norm and about 20 pointwise operations: fewer
than 200 roundings of 2^-24 relative to the largest intermediate of the output's kind, which the largest value of the output bounds within a
factor of 2 on these inputs (weights in 0.5 ... 1.5, means within 4 standard deviations of zero).  Sums over rows add (rows + 200) 2^-24 of the
sum of the magnitudes."""
import math

import pytest
import torch

from nmrf_amd import _lib
from nmrf_amd.ops import residual_norm

W = 2.0 ** -24
U = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NAMES = ("x", "y", "gate", "scale", "post_w", "post_b", "next_w", "next_b")


def formula(v, kind, post, nxt, act, scale_value, eps):
    def norm(z, w, b):
        if kind == "layer":
            z = z - z.mean(-1, keepdim=True)
        z = z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)
        z = z if w is None else z * w
        return z if b is None else z + b
    z = norm(v["y"], v["post_w"], v["post_b"]) if post else v["y"]
    if v["gate"] is not None:
        z = z * {None: lambda g: g, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[act](v["gate"])
    if v["scale"] is not None:
        z = z * v["scale"]
    out = v["x"] + scale_value * z
    return out, (norm(out, v["next_w"], v["next_b"]) if nxt else None)


def case(shape, dtype, kind="layer", gate=None, post=True, nxt=True, bias=True, scale=True, f32=False, seed=0, odd=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = shape[-1]

    def rand(shp, mean=0.0, std=1.0, dt=dtype):
        n = math.prod(shp)
        flat = torch.empty(n + 8, device="cuda", dtype=dt)
        v = flat[1 if odd else 0:][:n].view(shp)
        return v.copy_(torch.randn(shp, generator=gen, device="cuda") * std + mean)
    pt = torch.float32 if f32 else dtype
    bias = bias and kind == "layer"
    uni = lambda: (torch.rand(c, generator=gen, device="cuda") + 0.5).to(pt)  # noqa: E731
    v = {"x": rand(shape, 0.5, 2.0), "y": rand(shape, -0.3, 1.0), "gate": None if gate is None else rand(gate, 0.2, 0.7), "scale": uni() if scale else None,
         "post_w": uni() if post else None, "post_b": rand((c,), 0, 0.3, pt) if post and bias else None,
         "next_w": uni() if nxt else None, "next_b": rand((c,), 0, 0.3, pt) if nxt and bias else None}
    return v, rand(shape, 0.0, 0.3), (rand(shape, 0.0, 0.3) if nxt else None)


def run(v, d_out, d_h, kind, act, scale_value=None, eps=1e-5, grad=True, post=None, nxt=None):
    post = v["post_w"] is not None if post is None else post
    nxt = v["next_w"] is not None if nxt is None else nxt
    leaves = {k: None if t is None else t.detach().requires_grad_(grad) for k, t in v.items()}
    got = residual_norm(leaves["x"], leaves["y"], (leaves["next_w"], leaves["next_b"]) if nxt else None,
                        (leaves["post_w"], leaves["post_b"]) if post else None, leaves["gate"], act,
                        leaves["scale"] if leaves["scale"] is not None else scale_value, kind, eps)
    outs = got if nxt else (got,)
    if not grad:
        return outs, None
    pairs = [(o, d) for o, d in zip(outs, (d_out, d_h)) if d is not None]
    names = [k for k in NAMES if leaves[k] is not None]
    gr = torch.autograd.grad([o for o, _ in pairs], [leaves[k] for k in names], [d for _, d in pairs], allow_unused=True)
    return outs, dict(zip(names, gr))


def check(v, d_out, d_h, kind, act, scale_value=None, eps=1e-5):
    outs, grads = run(v, d_out, d_h, kind, act, scale_value, eps)
    post, nxt = v["post_w"] is not None, v["next_w"] is not None
    ref = {k: None if t is None else t.detach().double().requires_grad_(True) for k, t in v.items()}
    want = formula(ref, kind, post, nxt, act, 1.0 if scale_value is None else scale_value, eps)
    pairs = [(o, d.double()) for o, d in zip(want, (d_out, d_h)) if d is not None and o is not None]
    names = [k for k in NAMES if ref[k] is not None]
    wg = dict(zip(names, torch.autograd.grad([o for o, _ in pairs], [ref[k] for k in names], [d for _, d in pairs], allow_unused=True)))
    dtype, rows = v["x"].dtype, v["x"].numel() // v["x"].shape[-1]

    def near(a, b, what, room):
        assert a.shape == b.shape and a.dtype == (v[what].dtype if what in v else dtype), what
        tol = U[a.dtype] * b.abs() + room * W + (2.0 ** -25 if a.dtype == torch.float16 else 0)
        bad = (a.double() - b).abs() > tol
        assert not bool(bad.any()), (what, float((a.double() - b).abs().max()), float(room * W))
    for o, w, n in zip(outs, want, ("out", "h")):
        near(o, w.detach(), n, 400 * float(w.detach().abs().max()))
    for k in names:
        if wg[k] is None:
            assert grads[k] is None or not bool(grads[k].any()), k
            continue
        if k in ("x", "y") or (k == "gate" and v["gate"].numel() == v["x"].numel()):
            room = 400 * max(float(wg["x"].abs().max()) * (float(want[0].detach().abs().max()) if k == "gate" else 1.0), float(wg[k].abs().max()))
        else:                                                       # sums over rows and / or channels of products of O(1) factors
            terms = v["x"].shape[-1] if v[k].shape[-1] == 1 and k == "gate" else 1
            terms *= max(1, rows // max(1, v[k].numel() // (v[k].shape[-1])))
            room = (400 + terms) * math.sqrt(terms) * 8 * float(wg["x"].abs().max()) * max(3.0, float(want[0].detach().abs().max()))
        near(grads[k], wg[k], k, room)
    return outs, grads


# ---- refusals: on the host ------------------------------------------------------------------------------------------------------------
def test_refusals():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(_lib.NmrfHipError, match="MI355X only"):
        residual_norm(x, x)
    for kw, what in ((dict(kind="batch"), "kind"), (dict(gate_act="relu"), "gate_act"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps")):
        with pytest.raises(ValueError, match=what):
            residual_norm(x, x, **kw)
    with pytest.raises(ValueError, match="differ"):
        residual_norm(x, x[:1])
    with pytest.raises(ValueError, match="channels"):
        residual_norm(torch.zeros(2, 8193), torch.zeros(2, 8193))
    with pytest.raises(ValueError, match="channels"):
        residual_norm(torch.zeros(2, 0), torch.zeros(2, 0))


def test_c_entries_refuse_before_they_launch():
    lib = _lib.load()

    def fwd(x=64, y=64, t=4, c=8, dtype=0, kind=0, eps=1e-5, gate=None, rows=1, cols=1, act=0, out=64, h=64, pw=None, f32=0):
        return lib.nmrf_residual_norm(x, y, t, c, dtype, kind, eps, gate, rows, cols, act, 1.0, None, 1, pw, None, None, None, f32, out, h, None)
    assert fwd(t=0) == 0                                            # nothing to do
    assert fwd(x=None) == -3 and fwd(y=None) == -3 and fwd(out=None) == -3
    assert fwd(c=0) == -1 and fwd(c=8193) == -1 and fwd(t=-1) == -1 and fwd(dtype=3) == -1 and fwd(kind=2) == -1 and fwd(act=3) == -1
    assert fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1 and fwd(x=66) == -1 and fwd(x=65, dtype=1) == -1 and fwd(pw=66, f32=1, dtype=1) == -1
    assert fwd(gate=64, rows=3) == -1 and fwd(gate=64, rows=0) == -1 and fwd(gate=64, rows=2, cols=3) == -1

    def bwd(d_out=64, d_h=64, t=4, ws=64, floats=1 << 30, gate=None, rows=4, cols=1, dgate=None, post=1, dpw=None, dnw=None):
        return lib.nmrf_residual_norm_bwd(64, 64, d_out, d_h, t, 8, 0, 0, 1e-5, gate, rows, cols, 0, 1.0, None, post, None, None, None, 0, 64, 64,
                                          dgate, None, dpw, None, dnw, None, ws, floats, None)
    assert bwd(t=0) == -1 and bwd(ws=None) == -3 and bwd(d_out=None, d_h=None) == -3 and bwd(floats=8) == -1 and bwd(ws=66) == -1
    assert bwd(dgate=64) == -1 and bwd(d_h=None, dnw=64) == -1 and bwd(post=0, dpw=64) == -1 and bwd(gate=64, rows=3) == -1
    import ctypes
    n = ctypes.c_int64()
    assert lib.nmrf_residual_norm_bwd_size(4, 8, 3, ctypes.byref(n)) == -1 and lib.nmrf_residual_norm_bwd_size(4, 8, 2, None) == -3
    assert lib.nmrf_residual_norm_bwd_size(4, 8, 2, ctypes.byref(n)) == 0 and n.value >= 512 * 6 * 8


# ---- the formula ------------------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 1, 8), (2, 3, 128), (3, 5, 96), (2, 7, 100), (1, 65, 387), (2, 33, 512), (1, 9, 520), (1, 5, 2048), (1, 3, 2049),
          (2, 3, 4096), (1, 2, 5000), (1, 2, 8191), (1, 3, 8192), (4, 700, 64), (700, 3, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_row_layouts(shape, dtype):
    """Every layout of a row, with and without 16-byte loads, in both norms; gates and parameters vary along."""
    b, r, c = shape
    i = SHAPES.index(shape)
    gates = [None, (b, r, c), (b, r, 1), (b, 1, c), (b, 1, 1), (c,)]
    for j, kind in enumerate(("layer", "rms")):
        gate = gates[(i + j) % 6]
        v, d_out, d_h = case(shape, dtype, kind, gate, post=(i + j) % 3 != 2, f32=(i + j) % 2 == 1, seed=i, odd=i % 4 == 3)
        check(v, d_out, d_h, kind, (None, "sigmoid", "tanh")[(i + j) % 3] if gate is not None else None)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["element", "row", "sample", "sample_one", "channel", "one"])
@pytest.mark.parametrize("act", [None, "sigmoid", "tanh"])
def test_gates(gate, act):
    for shape in ((5, 41, 72), (2, 300, 256), (3, 2, 7, 48)):
        lead, c = shape[:-1], shape[-1]
        g = {"element": shape, "row": (*lead, 1), "sample": (lead[0],) + (1,) * (len(lead) - 1) + (c,), "sample_one": (lead[0],) + (1,) * len(lead),
             "channel": (c,), "one": (1,)}[gate]
        v, d_out, d_h = case(shape, torch.float32, "layer", g, seed=3)
        check(v, d_out, d_h, "layer", act)


@pytest.mark.gpu
@pytest.mark.parametrize("post,nxt,bias,scale", [(False, False, False, None), (True, False, True, 0.25), (False, True, False, True), (True, True, False, -1.5),
                                                 (True, True, True, True)])
def test_parts(post, nxt, bias, scale):
    for dtype in (torch.float32, torch.bfloat16):
        v, d_out, d_h = case((3, 50, 192), dtype, "layer", None, post, nxt, bias, scale is True, seed=4)
        check(v, d_out, d_h, "layer", None, None if scale is True else scale)
        if nxt:                                                     # either output alone
            check(v, d_out, None, "layer", None, None if scale is True else scale)
            check(v, None, d_h, "layer", None, None if scale is True else scale)


@pytest.mark.gpu
def test_norms_without_weights():
    v, d_out, d_h = case((4, 9, 64), torch.float32, "rms", None, seed=5, scale=False)
    for k in ("post_w", "post_b", "next_w", "next_b"):
        v[k] = None
    outs, grads = run(v, d_out, d_h, "rms", None, post=True, nxt=True)
    ref = {k: None if t is None else t.double().requires_grad_(True) for k, t in v.items()}
    want = formula(ref, "rms", True, True, None, 1.0, 1e-5)
    wg = torch.autograd.grad(want, (ref["x"], ref["y"]), (d_out.double(), d_h.double()))
    for a, b in zip((*outs, grads["x"], grads["y"]), (*want, *wg)):
        assert float((a.double() - b).abs().max()) <= 400 * W * float(b.abs().max())


@pytest.mark.gpu
def test_zero_rows_and_rows_that_are_constant():
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    out, h = residual_norm(x, x, (w, None), (w, None), scale=w)
    (out.sum() + h.sum()).backward()
    assert out.shape == (0, 16) and not bool(w.grad.any()) and x.grad.shape == (0, 16)
    v, d_out, d_h = case((2, 5, 64), torch.float32, seed=6)         # a row of one value: variance zero, held up by eps
    v["y"][0, 2] = 3.0
    v["y"][1] = 0.0
    check(v, d_out, d_h, "layer", None, eps=1e-3)
    check({**v, "post_b": None, "next_b": None}, d_out, d_h, "rms", None, eps=1e-3)


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_row():
    v, d_out, d_h = case((1, 64, 96), torch.float32, gate=(1, 64, 1), seed=7)
    clean, _ = run(v, d_out, d_h, "layer", "sigmoid", grad=False)
    v["y"][0, 3, 5], v["x"][0, 9, 0], v["gate"][0, 20, 0] = float("nan"), float("inf"), -float("inf")
    outs, grads = run(v, d_out, d_h, "layer", "sigmoid")
    keep = [i for i in range(64) if i not in (3, 9, 20)]
    assert all(torch.equal(o[:, keep], q[:, keep]) for o, q in zip(outs, clean))
    assert bool(torch.isnan(outs[0][0, 3]).all()) and bool(torch.isinf(outs[0][0, 9, 0])) and torch.equal(outs[0][0, 20], v["x"][0, 20])
    assert bool(torch.isfinite(grads["x"][:, keep]).all()) and float(grads["gate"][0, 20, 0].abs()) == 0.0


@pytest.mark.gpu
def test_drop_path_gate_keeps_dropped_samples_bit_for_bit():
    """Stochastic depth as the trunk of the Swin configuration applies it: a gate of 0 or 1 / keep for each sample."""
    v, d_out, d_h = case((6, 50, 96), torch.float32, scale=False, post=False, seed=8)
    v["gate"] = (torch.tensor([0, 1, 1, 0, 1, 0.0], device="cuda") / 0.75).view(6, 1, 1)
    outs, grads = check(v, d_out, d_h, "layer", None)
    assert torch.equal(outs[0][0], v["x"][0]) and not bool(grads["y"][3].any())


@pytest.mark.gpu
def test_gradients_against_differences_of_the_forward_pass():
    """Directional derivatives of L = <A, out> + <B, h> by central differences of the kernel at steps e and 2 e, extrapolated: (4 D(e) - D(2e)) / 3 is
    off by O(e^4).  L is summed in 64 bits from fp32 outputs whose errors (<= 100 * 2^-24 of O(4) values, N of them, random signs: sqrt(N)) are
    divided by e = 2^-5."""
    v, a, b = case((2, 20, 48), torch.float32, "layer", (2, 1, 48), seed=9)
    _, grads = run(v, a, b, "layer", "tanh")
    gen = torch.Generator(device="cuda").manual_seed(10)

    def loss(w):
        (out, h), _ = run(w, None, None, "layer", "tanh", grad=False)
        return float((out.double() * a.double()).sum() + (h.double() * b.double()).sum())
    for k in NAMES:
        d = torch.randn(v[k].shape, generator=gen, device="cuda")
        d = d / d.norm() * 2
        at = lambda e: loss({**v, k: v[k] + e * d})  # noqa: E731
        e = 2.0 ** -5
        dd = [(at(s * e) - at(-s * e)) / (2 * s * e) for s in (1, 2)]
        got = float((grads[k].double() * d.double()).sum())
        n = a.numel()
        room = 100 * W * 4 * math.sqrt(2 * n) * 0.3 / e * 2 + 2e-3 * abs(got) + 2e-4
        assert abs((4 * dd[0] - dd[1]) / 3 - got) <= room, (k, dd, got, room)


@pytest.mark.gpu
def test_repeats_streams_and_strides():
    v, d_out, d_h = case((3, 400, 320), torch.bfloat16, "rms", (3, 1, 320), seed=11)
    one = run(v, d_out, d_h, "rms", "sigmoid")
    two = run(v, d_out, d_h, "rms", "sigmoid")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        three = run(v, d_out, d_h, "rms", "sigmoid")
    torch.cuda.current_stream().wait_stream(s)
    t = lambda z: z.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731  (same values, other strides)
    four = run({**v, "x": t(v["x"]), "y": t(v["y"])}, t(d_out), d_h, "rms", "sigmoid")
    for other in (two, three, four):
        assert all(torch.equal(p, q) for p, q in zip(one[0], other[0])) and all(torch.equal(one[1][k], other[1][k]) for k in one[1])


@pytest.mark.gpu
def test_forward_is_captured_and_backward_refuses():
    v, d_out, d_h = case((2, 100, 256), torch.bfloat16, seed=12)
    call = lambda: residual_norm(v["x"], v["y"], (v["next_w"], v["next_b"]), (v["post_w"], v["post_b"]), scale=v["scale"])  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, h = call()
    for k in range(3):
        v["y"].mul_(-0.5)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(h, want[1])
    x = v["x"].clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(_lib.NmrfHipError, match="not captured"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(residual_norm(x, v["y"]), x, d_out)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_refusals_on_the_device():
    z = lambda *s, dt=torch.float32: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    x = z(2, 3, 8)
    with pytest.raises(_lib.NmrfHipError, match="fp32, bf16 or fp16"):
        residual_norm(x.double(), x.double())
    with pytest.raises(_lib.NmrfHipError, match="expected"):
        residual_norm(x, x.bfloat16())
    with pytest.raises(_lib.NmrfHipError, match="expected"):
        residual_norm(x, x, gate=z(2, 3, 1, dt=torch.bfloat16))
    for bad in ((2, 3, 4), (1, 3, 8), (3,), (2, 1, 3, 8), (2, 2, 1)):
        with pytest.raises(ValueError, match="gate"):
            residual_norm(x, x, gate=z(*bad))
    with pytest.raises(ValueError, match="post_weight"):
        residual_norm(x, x, post_norm=(z(7), None))
    with pytest.raises(_lib.NmrfHipError, match="all"):
        residual_norm(x.bfloat16(), x.bfloat16(), post_norm=(z(8), z(8, dt=torch.bfloat16)))
    with pytest.raises(_lib.NmrfHipError, match="contiguous"):
        residual_norm(x, x, post_norm=(z(16)[::2], None))
