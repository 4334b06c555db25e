"""What the training-block operators are measured on: an AdamW step over many tensors (moments in 32 or in 8 bits, the global gradient norm
clipped on the way), the norms around a block fused with its gate and residual scale, and the gated feed-forward block, with their
backward passes.

`own = False`: run() computes the plain forms (elementary torch operations in 32 bits, rounded once at the end).  `own = True`: run() makes
the calls a user of the framework makes (nmrf_amd.ops).  Both take what prepare() gives."""
import math

import torch

own = False

_DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_BLOCK = 256                                                        # values of a moment that share one scale in 8 bits
_LR, _B1, _B2, _EPS, _WD, _CLIP = 5e-4, 0.9, 0.999, 1e-8, 0.01, 1.0
_NORM_EPS = 1e-5


# ---- cases ----------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the stages of the stereo model itself: 15 message-passing layers at 128 channels, 180 tensors, stepped once per training step
        {"name": "adamw32 model", "op": "adamw", "bits": 32, "dtype": "fp32", "layers": 15, "dim": 128, "hidden": 512, "clip": True},
        # the same parameters with the moments in 8 bits
        {"name": "adamw8 model", "op": "adamw", "bits": 8, "dtype": "fp32", "layers": 15, "dim": 128, "hidden": 512, "clip": True},
        # a wide model in bf16: 202 million parameters, HBM-bound
        {"name": "adamw32 wide bf16", "op": "adamw", "bits": 32, "dtype": "bf16", "layers": 4, "dim": 2048, "hidden": 8192, "clip": True},
        # the same width in fp32 with 8-bit moments and no clipping
        {"name": "adamw8 wide", "op": "adamw", "bits": 8, "dtype": "fp32", "layers": 4, "dim": 2048, "hidden": 8192, "clip": False},
        # one token of a served model: latency
        {"name": "norm one token", "op": "norm", "kind": "rms", "dtype": "bf16", "batch": 1, "rows": 1, "channels": 4096, "post": True, "gate": "none",
         "gate_act": "none", "scale": True, "train": False},
        # the tokens of one KITTI frame (1/8 resolution, four labels a pixel) through a layer of the message passing, forward and backward
        {"name": "norm kitti train", "op": "norm", "kind": "layer", "dtype": "fp32", "batch": 1, "rows": 29952, "channels": 128, "post": False, "gate": "none",
         "gate_act": "none", "scale": True, "train": True},
        # a sandwich-normed wide layer with a gate for each sample (conditioned blocks, stochastic depth), forward and backward
        {"name": "norm wide train", "op": "norm", "kind": "rms", "dtype": "bf16", "batch": 8, "rows": 2048, "channels": 4096, "post": True, "gate": "sample",
         "gate_act": "tanh", "scale": True, "train": True},
        # odd channels and rows, a gate for each row
        {"name": "norm odd train", "op": "norm", "kind": "layer", "dtype": "fp16", "batch": 3, "rows": 1667, "channels": 387, "post": True, "gate": "row",
         "gate_act": "sigmoid", "scale": False, "train": True},
        # one token of a served model: the weights are read once
        {"name": "ffn one token", "op": "ffn", "dtype": "bf16", "rows": 1, "dim": 4096, "hidden": 11008, "act": "silu", "bias": False, "train": False},
        # the tokens of one KITTI frame at the message passing's width, forward and backward
        {"name": "ffn kitti train", "op": "ffn", "dtype": "fp32", "rows": 29952, "dim": 128, "hidden": 512, "act": "gelu", "bias": True, "train": True},
        # a wide layer over a long batch of tokens, forward and backward
        {"name": "ffn wide train", "op": "ffn", "dtype": "bf16", "rows": 8192, "dim": 2048, "hidden": 5504, "act": "silu", "bias": False, "train": True},
        # sizes that fit no tile
        {"name": "ffn odd train", "op": "ffn", "dtype": "fp16", "rows": 777, "dim": 321, "hidden": 861, "act": "silu", "bias": True, "train": True},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["adamw", "norm", "ffn"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "adamw":
        dim = _spread(rng, 24, 1024)
        return {"op": op, "bits": rng.choice([32, 8]), "dtype": dtype, "layers": rng.randint(1, 15), "dim": dim, "hidden": dim * 2 + rng.randint(0, 2 * dim),
                "clip": rng.random() < 0.7}
    if op == "norm":
        channels = _spread(rng, 16, 4096)
        batch = rng.randint(1, 8)
        return {"op": op, "kind": rng.choice(["layer", "rms"]), "dtype": dtype, "batch": batch, "rows": max(1, _spread(rng, 1, 30000) * 128 // max(128, channels)),
                "channels": channels, "post": rng.random() < 0.6, "gate": rng.choice(["none", "full", "row", "sample"]),
                "gate_act": rng.choice(["none", "sigmoid", "tanh"]), "scale": rng.random() < 0.5, "train": rng.random() < 0.7}
    dim = _spread(rng, 32, 2048)
    return {"op": op, "dtype": dtype, "rows": max(1, min(_spread(rng, 1, 30000), 8192 * 1024 // dim)), "dim": dim, "hidden": dim * 2 + rng.randint(0, dim // 2),
            "act": rng.choice(["silu", "gelu", "relu"]), "bias": rng.random() < 0.5, "train": rng.random() < 0.6}


# ---- inputs -----------------------------------------------------------------------------------------------------------------------
def _shapes(case):
    """Matrices first (they decay), then vectors (they do not): the tensors of `layers` message-passing layers."""
    c, f = case["dim"], case["hidden"]
    return [(3 * c, c + 31), (c, c), (f, c), (c, f)] * case["layers"], [(3 * c,), (c,), (f,), (c,), (c,), (c,), (c,), (c,)] * case["layers"]


def _starts(shapes):
    """Where each tensor begins in the flat buffers: at multiples of a block, so that a block never holds two tensors."""
    at, total = [], 0
    for s in shapes:
        at.append(total)
        total += -(-math.prod(s) // _BLOCK) * _BLOCK
    return at, total


def _views(flat, shapes, at):
    return [flat[a:a + math.prod(s)].view(s) for s, a in zip(shapes, at)]


def _prepare_adamw(case, gen):
    mats, vecs = _shapes(case)
    shapes = mats + vecs
    at, total = _starts(shapes)
    dtype = _TYPES[case["dtype"]]
    used = torch.zeros(total, device=_DEVICE, dtype=torch.bool)
    for s, a in zip(shapes, at):
        used[a:a + math.prod(s)] = True
    normal = lambda std: torch.randn(total, generator=gen, device=_DEVICE, dtype=torch.float32).mul_(std).mul_(used)  # noqa: E731
    # gradients of a mean loss: small, and of a different size in every tensor
    size = torch.exp(torch.randn(len(shapes), generator=gen, device=_DEVICE) - 5.0)
    ends = torch.tensor(at[1:] + [total], device=_DEVICE)
    grad = normal(1.0)
    grad.mul_(size.repeat_interleave(torch.diff(ends, prepend=ends.new_zeros(1)))[:total])
    s = {"case": case, "shapes": shapes, "at": at, "total": total, "split": at[len(mats)], "step": 0, "seed": 1234,
         "p": normal(0.05).to(dtype), "g": grad.to(dtype), "decay": [_WD] * len(mats) + [0.0] * len(vecs)}
    s["params"], s["grads"] = _views(s["p"], shapes, at), _views(s["g"], shapes, at)
    if case["bits"] == 32:
        for k in ("m", "v"):
            s[k] = torch.zeros(total, device=_DEVICE, dtype=torch.float32)
            s[k + "s"] = _views(s[k], shapes, at)
    else:
        for k in ("m", "v"):
            s[k] = torch.zeros(total, device=_DEVICE, dtype=torch.uint8)
            s[k + "_scale"] = torch.zeros(total // _BLOCK, device=_DEVICE, dtype=torch.float32)
            s[k + "s"] = _views(s[k], shapes, at)
            s[k + "_scales"] = [s[k + "_scale"][a // _BLOCK:a // _BLOCK + -(-math.prod(x) // _BLOCK)] for x, a in zip(shapes, at)]
    return s


def _prepare_norm(case, gen):
    b, r, c, dtype = case["batch"], case["rows"], case["channels"], _TYPES[case["dtype"]]
    rand = lambda *shape, std=1.0, mean=0.0: (torch.randn(*shape, generator=gen, device=_DEVICE) * std + mean).to(dtype)  # noqa: E731
    s = {"case": case, "x": rand(b, r, c, std=2.0), "y": rand(b, r, c), "next_w": rand(c, std=0.1, mean=1.0)}
    s["next_b"] = rand(c, std=0.1) if case["kind"] == "layer" else None
    s["post_w"] = rand(c, std=0.1, mean=1.0) if case["post"] else None
    s["post_b"] = rand(c, std=0.1) if case["post"] and case["kind"] == "layer" else None
    s["gate"] = {"none": None, "full": rand(b, r, c), "row": rand(b, r, 1), "sample": rand(b, 1, c)}[case["gate"]] if case["gate"] != "none" else None
    s["scale"] = rand(c, std=0.05, mean=0.5) if case["scale"] else None
    if case["train"]:
        s["d_out"], s["d_h"] = rand(b, r, c, std=0.01), rand(b, r, c, std=0.01)
    return s


def _prepare_ffn(case, gen):
    t, d, f, dtype = case["rows"], case["dim"], case["hidden"], _TYPES[case["dtype"]]
    rand = lambda *shape, std=1.0: (torch.randn(*shape, generator=gen, device=_DEVICE) * std).to(dtype)  # noqa: E731
    s = {"case": case, "x": rand(t, d), "w_gate": rand(f, d, std=d ** -0.5), "w_up": rand(f, d, std=d ** -0.5), "w_down": rand(d, f, std=f ** -0.5)}
    s["b_gate"], s["b_up"], s["b_down"] = (rand(f, std=0.1), rand(f, std=0.1), rand(d, std=0.1)) if case["bias"] else (None, None, None)
    if case["train"]:
        s["dy"] = rand(t, d, std=0.01)
    return s


_INPUTS = {"norm": ("x", "y", "gate", "scale", "post_w", "post_b", "next_w", "next_b"),
           "ffn": ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")}


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE)
    gen.manual_seed(int(seed))
    s = {"adamw": _prepare_adamw, "norm": _prepare_norm, "ffn": _prepare_ffn}[case["op"]](case, gen)
    if case.get("train"):                                           # what a training program differentiates: parameters and activations
        for k in _INPUTS[case["op"]]:
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------------
def _random32(index, key):
    """32 random bits of (element index, key): a Weyl step by the golden ratio and two rounds of xor-shift and odd multiplication."""
    mask = 0xFFFFFFFF
    x = (index * 0x9E3779B9 + key) & mask
    x = ((x ^ (x >> 16)) * 0x6C62272D) & mask
    x = ((x ^ (x >> 15)) * 0x2C9277B5) & mask
    return x ^ (x >> 16)


def _encode(a, mantissa, rnd):
    """|values| of [blocks, 256] in 3 exponent and `mantissa` mantissa bits under a power-of-two scale, rounded up with the probability of the
    dropped fraction (`rnd`: as many random bits as are dropped).  -> (codes, scales)"""
    drop = 23 - mantissa
    top = a.amax(-1, keepdim=True)
    scale = torch.where(top >= 2.0 ** -100, (top.view(torch.int32) & 0x7F800000).view(torch.float32), torch.zeros_like(top))
    x = a * torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    normal = ((x.view(torch.int32) + rnd) >> drop) - (120 << mantissa)
    small = ((x * 2.0 ** 29).to(torch.int32) + rnd) >> drop
    code = torch.where(x >= 2.0 ** -6, normal, small)
    return code.clamp_(max=(8 << mantissa) - 1), scale


def _decode(code, mantissa, scale):
    field, man = code >> mantissa, code & ((1 << mantissa) - 1)
    normal = ((field + 120) << 23 | man << (23 - mantissa)).view(torch.float32)
    return torch.where(field > 0, normal, man.to(torch.float32) * 2.0 ** (-6 - mantissa)) * scale


def _moments(s):
    """The 8-bit moments as the values they stand for: [blocks, 256] m and sqrt(v)."""
    mc, vc = s["m"].view(-1, _BLOCK).to(torch.int32), s["v"].view(-1, _BLOCK).to(torch.int32)
    m = _decode(mc & 127, 4, s["m_scale"][:, None])
    return torch.where(mc > 127, -m, m), _decode(vc, 5, s["v_scale"][:, None])


def _plain_adamw(s):
    case, t = s["case"], s["step"]
    g = s["g"].float()
    out = {}
    if case["clip"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * (_CLIP / (norm + 1e-6)).clamp(max=1.0)
        out["norm"] = norm
    if case["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m, r = (x.view(-1) for x in _moments(s))
        v = r * r
    m = m * _B1 + g * (1 - _B1)
    v = v * _B2 + (g * g) * (1 - _B2)
    r = v.double().sqrt().float()                                   # (correctly rounded: its 8-bit code is decided next to borders)
    p = s["p"].float()
    p = torch.cat((p[:s["split"]] * (1 - _LR * _WD), p[s["split"]:]))
    p = p - (m * (_LR / (1 - _B1 ** t))) / (r * (1 / math.sqrt(1 - _B2 ** t)) + _EPS)
    s["p"].copy_(p)
    out["p"] = s["p"]
    if case["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {**out, "m": s["m"], "v": s["v"]}
    at = torch.tensor(s["at"], device=p.device)
    count = torch.diff(at, append=at.new_tensor([s["total"]]))
    index = torch.arange(s["total"], device=p.device) - at.repeat_interleave(count)
    key = (torch.arange(len(s["at"]), device=p.device) * 0x85157AF5 + s["seed"] * 0x9E3779B1 + t * 0xC2B2AE3D) & 0xFFFFFFFF
    rnd = _random32(index, key.repeat_interleave(count)).view(-1, _BLOCK)
    m = m.view(-1, _BLOCK)
    code, scale = _encode(m.abs(), 4, (rnd >> 18 << 5).to(torch.int32))
    s["m"].copy_((code | (m < 0).to(torch.int32) << 7).view(-1))
    s["m_scale"].copy_(scale.view(-1))
    r = r.view(-1, _BLOCK)
    code, scale = _encode(r, 5, (rnd & 0x3FFFF).to(torch.int32))
    s["v"].copy_(torch.where((r > 0) & (scale > 0), code.clamp(min=1), code).view(-1))
    s["v_scale"].copy_(scale.view(-1))
    m, r = _moments(s)
    return {**out, "m": m.view(-1), "v": (r * r).view(-1)}


def _norm(z, kind):
    if kind == "layer":
        z = z - z.mean(-1, keepdim=True)
    rstd = (z.square().mean(-1, keepdim=True) + _NORM_EPS).rsqrt()
    return z * rstd, rstd


def _norm_back(u, zhat, rstd, kind):
    inner = zhat * (u * zhat).mean(-1, keepdim=True)
    return rstd * (u - inner - (u.mean(-1, keepdim=True) if kind == "layer" else 0.0))


def _affine(z, w, b):
    return z * w.float() if b is None else z * w.float() + b.float()


def _plain_norm(s):
    case, kind = s["case"], s["case"]["kind"]
    x, y, dtype = s["x"].detach().float(), s["y"].detach().float(), s["x"].dtype
    zhat, zrstd = _norm(y, kind) if case["post"] else (None, None)
    z = _affine(zhat, s["post_w"].detach(), None if s["post_b"] is None else s["post_b"].detach()) if case["post"] else y
    act = {"none": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[case["gate_act"]]
    gate = act(s["gate"].detach().float()) if s["gate"] is not None else None
    f = None if gate is None else gate
    if s["scale"] is not None:
        f = s["scale"].detach().float() if f is None else f * s["scale"].detach().float()
    out = x + (z if f is None else f * z)
    hhat, hrstd = _norm(out, kind)
    h = _affine(hhat, s["next_w"].detach(), None if s["next_b"] is None else s["next_b"].detach())
    got = {"out": out.to(dtype), "h": h.to(dtype)}
    if not case["train"]:
        return got
    rows = (0, 1)
    dh = s["d_h"].float()
    got["d_next_w"] = (dh * hhat).sum(rows).to(dtype)
    if kind == "layer":
        got["d_next_b"] = dh.sum(rows).to(dtype)
    dx = s["d_out"].float() + _norm_back(dh * s["next_w"].detach().float(), hhat, hrstd, kind)
    got["d_x"] = dx.to(dtype)
    dz = dx if f is None else dx * f
    if s["scale"] is not None:
        got["d_scale"] = (dx * z if gate is None else dx * z * gate).sum(rows).to(dtype)
    if gate is not None:
        dgate = dx * z if s["scale"] is None else dx * z * s["scale"].detach().float()
        dgate = dgate if case["gate"] == "full" else dgate.sum(-1, keepdim=True) if case["gate"] == "row" else dgate.sum(1, keepdim=True)
        slope = {"none": lambda v: 1.0, "sigmoid": lambda v: v * (1 - v), "tanh": lambda v: 1 - v * v}[case["gate_act"]](gate)
        got["d_gate"] = (dgate * slope).to(dtype)
    if case["post"]:
        got["d_post_w"] = (dz * zhat).sum(rows).to(dtype)
        if kind == "layer":
            got["d_post_b"] = dz.sum(rows).to(dtype)
        dz = _norm_back(dz * s["post_w"].detach().float(), zhat, zrstd, kind)
    got["d_y"] = dz.to(dtype)
    return got


def _act_and_slope(g, act):
    if act == "relu":
        on = (g > 0).float()
        return g * on, on
    if act == "silu":
        sig = torch.sigmoid(g)
        return g * sig, sig * (1 + g * (1 - sig))
    phi = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
    return g * phi, phi + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5


def _plain_ffn(s):
    case, dtype = s["case"], s["x"].dtype
    v = {k: None if s[k] is None else s[k].detach().float() for k in _INPUTS["ffn"]}
    g, u = v["x"] @ v["w_gate"].t(), v["x"] @ v["w_up"].t()
    if case["bias"]:
        g, u = g + v["b_gate"], u + v["b_up"]
    a, slope = _act_and_slope(g, case["act"])
    h = a * u
    y = h @ v["w_down"].t()
    got = {"y": (y + v["b_down"] if case["bias"] else y).to(dtype)}
    if not case["train"]:
        return got
    dy = s["dy"].float()
    dh = dy @ v["w_down"]
    du, dg = dh * a, dh * u * slope
    got["d_x"] = (dg @ v["w_gate"] + du @ v["w_up"]).to(dtype)
    got["d_w_gate"], got["d_w_up"], got["d_w_down"] = (dg.t() @ v["x"]).to(dtype), (du.t() @ v["x"]).to(dtype), (dy.t() @ h).to(dtype)
    if case["bias"]:
        got["d_b_gate"], got["d_b_up"], got["d_b_down"] = dg.sum(0).to(dtype), du.sum(0).to(dtype), dy.sum(0).to(dtype)
    return got


# ---- the framework's calls --------------------------------------------------------------------------------------------------------
def _own_adamw(s):
    from nmrf_amd import ops
    case = s["case"]
    if "plan" not in s:                                             # kept beside the moments for the whole training run
        scales = () if case["bits"] == 32 else (s["m_scales"], s["v_scales"])
        s["plan"] = ops.AdamWPlan(s["params"], s["ms"], s["vs"], *scales, weight_decay=s["decay"])
    norm = s["plan"].step(s["grads"], step=s["step"], lr=_LR, betas=(_B1, _B2), eps=_EPS, max_norm=_CLIP if case["clip"] else None, seed=s["seed"])
    out = {"norm": norm, "p": s["p"]} if case["clip"] else {"p": s["p"]}
    if case["bits"] == 32:
        return {**out, "m": s["m"], "v": s["v"]}
    return {**out, "m": ops.adamw_moment(s["m"], s["m_scale"]), "v": ops.adamw_moment(s["v"], s["v_scale"], squared=True)}


def _gradients(out, grads, s, names):
    names = [k for k in names if s[k] is not None]
    return {"d_" + k: v for k, v in zip(names, torch.autograd.grad(out, [s[k] for k in names], grads))}


def _own_norm(s):
    from nmrf_amd import ops
    case = s["case"]
    post = (s["post_w"], s["post_b"]) if case["post"] else None
    out, h = ops.residual_norm(s["x"], s["y"], next_norm=(s["next_w"], s["next_b"]), post_norm=post, gate=s["gate"],
                               gate_act=None if case["gate_act"] == "none" else case["gate_act"], scale=s["scale"], kind=case["kind"], eps=_NORM_EPS)
    got = {"out": out.detach(), "h": h.detach()}
    return got if not case["train"] else {**got, **_gradients((out, h), (s["d_out"], s["d_h"]), s, _INPUTS["norm"])}


def _own_ffn(s):
    from nmrf_amd import ops
    y = ops.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["b_gate"], s["b_up"], s["b_down"], act=s["case"]["act"])
    got = {"y": y.detach()}
    return got if not s["case"]["train"] else {**got, **_gradients((y,), (s["dy"],), s, _INPUTS["ffn"])}


def run(state):
    op = state["case"]["op"]
    if op == "adamw":
        state["step"] += 1
    if own:
        return {"adamw": _own_adamw, "norm": _own_norm, "ffn": _own_ffn}[op](state)
    return {"adamw": _plain_adamw, "norm": _plain_norm, "ffn": _plain_ffn}[op](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------
def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "adamw":
        n = sum(math.prod(s) for part in _shapes(case) for s in part)
        # p in and out, g in; the moments in and out, and in 8 bits (with a scale for each block) once more as the values that run() returns
        state = 16 if case["bits"] == 32 else 4 + 4 * 4 / _BLOCK + 8
        return {"bytes": n * (3 * e + state), "flops": 15 * n}
    if case["op"] == "norm":
        t, c = case["batch"] * case["rows"], case["channels"]
        gate = {"none": 0, "full": t * c, "row": t, "sample": case["batch"] * c}[case["gate"]]
        n = 4 * t * c + gate                                        # x, y in; out, h out
        if case["train"]:
            n += 6 * t * c + 2 * gate                               # the gradients of both outputs, out and y again; dx, dy out
        vectors = c * ((2 if case["kind"] == "layer" else 1) * (2 if case["post"] else 1) + (1 if case["scale"] else 0))
        return {"bytes": (n + vectors * (2 if case["train"] else 1)) * e, "flops": 20 * t * c * (3 if case["train"] else 1)}
    t, d, f = case["rows"], case["dim"], case["hidden"]
    products = 6 * t * d * f * (3 if case["train"] else 1)
    return {"bytes": (2 * t * d + 3 * d * f + ((2 * t * d + 3 * d * f) if case["train"] else 0)) * e, "flops": products}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------
def _exact_adamw(case, seed):
    s = prepare(case, seed)
    g, p, out = s["g"].double(), s["p"].double(), {}
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, _CLIP / (float(out["norm"]) + 1e-6))
    m, v = (1 - _B1) * g, (1 - _B2) * g ** 2                        # the first step from moments of zero
    decay = torch.full_like(p, _LR * _WD)
    decay[s["split"]:] = 0
    out["p"] = p * (1 - decay) - _LR * (m / (1 - _B1)) / ((v / (1 - _B2)) ** 0.5 + _EPS)
    # (a moment in 8 bits jumps by a whole step where the last bit before it crosses a border: no value in 64 bits to hold it to)
    return {**out, "m": m, "v": v} if case["bits"] == 32 else {**out, "m": None, "v": None}


def _definition_norm(z, weight, bias, kind):
    mean = z.mean(-1, keepdim=True) if kind == "layer" else 0.0
    z = (z - mean) / torch.sqrt(((z - mean) ** 2).mean(-1, keepdim=True) + _NORM_EPS) * weight
    return z if bias is None else z + bias


def exact(case, seed):
    """What run() returns for these inputs, from the definitions in 64 bits: the gradients by differentiating the forward formula."""
    if case["op"] == "adamw":
        return _exact_adamw(case, seed)
    s = prepare(case, seed)
    names = [k for k in _INPUTS[case["op"]] if s[k] is not None]
    v = {k: s[k].detach().double().requires_grad_(case["train"]) for k in names}
    if case["op"] == "norm":
        z = _definition_norm(v["y"], v["post_w"], v.get("post_b"), case["kind"]) if case["post"] else v["y"]
        if "gate" in v:
            z = z * {"none": lambda q: q, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[case["gate_act"]](v["gate"])
        out = v["x"] + (z * v["scale"] if "scale" in v else z)
        h = _definition_norm(out, v["next_w"], v.get("next_b"), case["kind"])
        outs, grads, got = (out, h), ("d_out", "d_h"), {"out": out.detach(), "h": h.detach()}
    else:
        g, u = v["x"] @ v["w_gate"].T, v["x"] @ v["w_up"].T
        if case["bias"]:
            g, u = g + v["b_gate"], u + v["b_up"]
        a = {"relu": torch.relu, "silu": lambda q: q / (1 + torch.exp(-q)), "gelu": lambda q: q * torch.special.ndtr(q)}[case["act"]](g)
        y = (a * u) @ v["w_down"].T
        y = y + v["b_down"] if case["bias"] else y
        outs, grads, got = (y,), ("dy",), {"y": y.detach()}
    if case["train"]:
        got.update(zip(["d_" + k for k in names], torch.autograd.grad(outs, [v[k] for k in names], [s[k].double() for k in grads])))
    return got
