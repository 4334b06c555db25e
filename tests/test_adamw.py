"""AdamW over many tensors with 32- and 8-bit moments (csrc/adamw.hip, nmrf_amd/ops/adamw.py, nmrf_amd/optim.py) against the formula in
64 bits, and -- where codes of 8 bits are decided -- against the same roundings written in torch."""
import ctypes
import math

import numpy as np
import pytest
import torch

from nmrf_amd import _lib
from nmrf_amd import optim as O
from nmrf_amd.ops import AdamWPlan, adamw_moment

LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.99, 1e-8, 0.1
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SIZES = [1, 3, 0, 255, 256, 257, 4095, 4096, 4097, 16384, 16385, 70001, 1024]


# ---- refusals: on the host, no GPU ----------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    p = [torch.zeros(8)]
    with pytest.raises(_lib.NmrfHipError, match="MI355X only"):
        AdamWPlan(p, [torch.zeros(8)], [torch.zeros(8)])
    q = torch.nn.Parameter(torch.zeros(8))
    q.grad = torch.zeros(8)
    with pytest.raises(_lib.NmrfHipError, match="MI355X only"):
        O.AdamW([q]).step()


def test_arguments_are_refused():
    with pytest.raises(ValueError, match="no parameters"):
        AdamWPlan([], [], [])
    with pytest.raises(_lib.NmrfHipError, match="fp32, bf16 or fp16"):
        AdamWPlan([torch.zeros(4, dtype=torch.float64)], [torch.zeros(4)], [torch.zeros(4)])
    with pytest.raises(ValueError, match="lists of"):
        AdamWPlan([torch.zeros(4)], [], [torch.zeros(4)])
    p = [torch.nn.Parameter(torch.zeros(4))]
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            O.AdamW(p, **bad)
    with pytest.raises(ValueError, match="max_norm"):
        O.AdamW(p).step(max_norm=0.0)
    assert O.AdamW(p).step(max_norm=1.0) is None                    # no gradients: nothing to do


def test_c_entry_refuses_before_it_launches():
    lib = _lib.load()
    a = lambda *v: np.array(v, np.uint64)  # noqa: E731
    keep, at = [], lambda x: keep.append(x) or x.ctypes.data  # noqa: E731
    numel, hyper, betas = np.array([4, 4], np.int64), np.zeros(8, np.float32), np.zeros(4, np.float32)

    def call(p, g=a(16, 32), m=a(48, 64), v=a(80, 96), dtype=0, bits=32, n=2, ms=None, vs=None, key=None):
        return lib.nmrf_adamw_step(n, at(p), at(g), at(m), at(v), ms, vs, numel.ctypes.data, hyper.ctypes.data, key, betas.ctypes.data, dtype, bits,
                                   None, None)
    assert call(a(112, 112)) == -1                                  # one parameter twice
    assert call(a(112, 0)) == -3                                    # null
    assert call(a(112, 130)) == -1                                  # not aligned to its type
    assert call(a(112, 128), dtype=3) == -1 and call(a(112, 128), bits=16) == -1 and call(a(112, 128), n=0) == -1
    assert call(a(112, 128), bits=8) == -3                          # 8 bits without scales
    numel[0] = -1
    assert call(a(112, 128)) == -1
    numel[0] = 4
    parts = np.zeros(1)
    assert lib.nmrf_grad_sqsum(2, at(a(16, 32)), numel.ctypes.data, 0, 64, 1, None) == -1            # two partials, room for one
    assert lib.nmrf_grad_sqsum(2, at(a(16, 33)), numel.ctypes.data, 0, 64, 2, None) == -1
    assert lib.nmrf_grad_norm(parts.ctypes.data, 0, ctypes.c_float(1.0), 64, None) == -1
    assert lib.nmrf_grad_norm(parts.ctypes.data, 1, ctypes.c_float(0.0), 64, None) == -1
    assert lib.nmrf_grad_norm(parts.ctypes.data, 1, ctypes.c_float(float("nan")), 64, None) == -1
    assert lib.nmrf_adamw_moment_f32(None, 64, 1, 0, 64, None) == -3 and lib.nmrf_adamw_moment_f32(64, 64, 0, 0, 64, None) == -1


def test_state_dict_is_torchs_and_other_bits_are_refused():
    p = [torch.nn.Parameter(torch.randn(5000)), torch.nn.Parameter(torch.randn(3))]
    t = torch.optim.AdamW([{"params": p[:1], "lr": 1e-3}, {"params": p[1:], "lr": 1e-4, "weight_decay": 0.0}])
    for q in p:
        q.grad = torch.randn_like(q)
    t.step()
    o = O.AdamW([{"params": p[:1]}, {"params": p[1:]}])
    o.load_state_dict(t.state_dict())
    assert [g["lr"] for g in o.param_groups] == [1e-3, 1e-4] and o.state[p[0]]["step"] == 1
    back = torch.optim.AdamW([{"params": p[:1]}, {"params": p[1:]}])
    back.load_state_dict(o.state_dict())
    assert float(back.state[p[1]]["step"]) == 1.0 and torch.equal(back.state[p[0]]["exp_avg"], t.state[p[0]]["exp_avg"])
    back.step()                                                     # (the steps of a loaded state are tensors of their own)
    assert float(back.state[p[1]]["step"]) == 2.0 and o.state[p[1]]["step"] == 1
    with pytest.raises(ValueError, match="8"):
        O.AdamW([{"params": p[:1]}, {"params": p[1:]}], state_bits=8).load_state_dict(t.state_dict())
    with pytest.raises(ValueError, match="parameter groups"):
        O.AdamW(p).load_state_dict(t.state_dict())


def test_optimizer_is_copied_with_its_settings():
    import copy
    o = O.AdamW([torch.nn.Parameter(torch.zeros(4))], lr=0.5, state_bits=8, min_8bit_size=7, seed=3)
    c = copy.deepcopy(o)
    assert (c.state_bits, c.min_8bit_size, c.seed, c.param_groups[0]["lr"]) == (8, 7, 3, 0.5) and c.step() is None


# ---- the formula ----------------------------------------------------------------------------------------------------------------------
def _case(sizes, dtype, bits, seed, odd=False):
    """Parameters, gradients and moments as views of storage with sentinels between them (odd: none of them aligned to 16 bytes)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lead = 1 if odd else 16

    def views(dt, fill=None, std=1.0, ns=sizes):
        total = sum(-(-n // 16) * 16 + 32 for n in ns) + 32
        flat = torch.full((total,), 77, device="cuda", dtype=torch.float32).to(dt)
        at, out = lead, []
        for n in ns:
            v = flat[at:at + n]
            v.copy_(torch.randn(n, generator=gen, device="cuda") * std if fill is None else torch.full((n,), fill, device="cuda"))
            out.append(v)
            at += -(-n // 16) * 16 + 32
        keep = torch.ones(total, dtype=torch.bool, device="cuda")
        for v in out:
            keep[v.storage_offset():v.storage_offset() + v.numel()] = False
        return out, lambda: bool((flat[keep].float() == 77).all())
    p, okp = views(dtype)
    g, okg = views(dtype, std=1e-2)
    st = torch.float32 if bits == 32 else torch.uint8
    m, okm = views(st, fill=0)
    v, okv = views(st, fill=0)
    blocks = [-(-n // 256) for n in sizes]
    sm, oks = views(torch.float32, fill=0, ns=blocks) if bits == 8 else (None, lambda: True)
    sv, okt = views(torch.float32, fill=0, ns=blocks) if bits == 8 else (None, lambda: True)
    return p, g, m, v, sm, sv, lambda: all(f() for f in (okp, okg, okm, okv, oks, okt))


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_steps_in_32_bits(dtype, odd):
    sizes = SIZES * 17                                              # 221 tensors: several launches of both kernels
    p, g, m, v, _, _, intact = _case(sizes, dtype, 32, 3, odd)
    decay = [WD * (i % 3) for i in range(len(sizes))]
    plan = AdamWPlan(p, m, v, weight_decay=decay)
    pd, md, vd = ([x.double() for x in t] for t in (p, m, v))
    u, w = U[dtype], 2.0 ** -24
    for t in range(1, 4):
        gd = [x.double() for x in g]
        total = math.sqrt(sum(float((x * x).sum()) for x in gd))
        norm = plan.step(g, step=t, lr=LR, betas=(B1, B2), eps=EPS, max_norm=0.5)
        c = min(1.0, 0.5 / (total + 1e-6))
        assert abs(float(norm) - total) <= 2 * w * total
        for i in range(len(sizes)):
            gc = gd[i] * c
            # one step from what the kernel holds: roundings per operation (constants rounded to fp32 count as one each, c as three)
            a, b = B1 * md[i], (1 - B1) * gc
            em = w * (4 * a.abs() + 7 * b.abs())
            md[i] = a + b
            a2, b2 = B2 * vd[i], (1 - B2) * gc * gc
            ev = w * (4 * a2 + 12 * b2)
            vd[i] = a2 + b2
            assert bool(((m[i].double() - md[i]).abs() <= em + 1e-44).all()) and bool(((v[i].double() - vd[i]).abs() <= ev + 1e-44).all())
            md[i], vd[i] = m[i].double(), v[i].double()             # (their error is judged above: the update from the moments as they are)
            up = LR / (1 - B1 ** t) * md[i] / (vd[i].sqrt() / math.sqrt(1 - B2 ** t) + EPS)
            want = pd[i] * (1 - LR * decay[i]) - up
            # 1 - lr wd rounded, product, difference: 3 roundings of p; the update: constant, product, root, constant, product, sum, quotient
            assert bool(((p[i].double() - want).abs() <= (u if dtype != torch.float32 else 0) * want.abs() * (1 + u) + w * (3 * pd[i].abs() + 9 * up.abs())
                         + (6e-8 if dtype == torch.float16 else 0)).all())
            pd[i] = p[i].double()
        for x in g:
            x.mul_(0.5)
    assert intact()


def _pow2(e):
    """2^e in 64 bits from its bits (torch.ldexp goes through pow, which is not exact for every whole exponent)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _mirror8(p, g, c, mcode, ms, vcode, vs, t, decay, key):
    """The step on [blocks, 256] fp32 tensors with every operation rounded as the kernel documents it; codes and scales by its rules."""
    def dec(code, man, scale):
        e, f = code >> man, code & ((1 << man) - 1)
        return torch.where(e > 0, (1 + f.double() / (1 << man)) * _pow2(e - 7), f.double() / (64 << man)).float() * scale[:, None]

    def enc(a, man, rnd, bits):
        top = a.amax(-1, keepdim=True)
        scale = torch.where(top >= 2.0 ** -100, _pow2(torch.frexp(top)[1] - 1).float(), torch.zeros_like(top))
        x = torch.where(scale > 0, a.double() / scale.double().clamp(min=1e-300), torch.zeros_like(a.double()))
        e = (torch.frexp(x)[1] - 1).clamp(min=-6)
        # the kernel adds the random bits to the dropped bits of the float (subnormals: of x 2^29, truncated) and cuts
        grid = torch.where(x >= 2.0 ** -6, torch.floor(x * _pow2(23 - e)), torch.floor(x * 2.0 ** 29))
        q = torch.floor((grid + rnd.double()) / 2.0 ** bits) * _pow2(e - man)
        q = q.clamp(max=2 - 2.0 ** -man)
        e2 = (torch.frexp(q)[1] - 1).clamp(min=-6)
        code = torch.where(q >= 2.0 ** -6, (e2 + 7 << man) + (q * _pow2(-e2) - 1) * (1 << man), q * (64 << man)).long()
        return code, scale.squeeze(-1)
    m = dec(mcode & 127, 4, ms)
    m = torch.where(mcode > 127, -m, m)
    r = dec(vcode, 5, vs)
    v = r * r
    g = g * c
    m = m * B1 + g * (1 - B1)
    v = v * B2 + (g * g) * (1 - B2)
    r = v.double().sqrt().float()
    p = p * (1 - LR * decay) - (m * (LR / (1 - B1 ** t))) / (r * (1 / math.sqrt(1 - B2 ** t)) + EPS)
    i = torch.arange(m.numel(), device=m.device).view(m.shape)
    x = (i * 0x9E3779B9 + key) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x6C62272D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x2C9277B5) & 0xFFFFFFFF
    x = x ^ (x >> 16)
    mc, msc = enc(m.abs(), 4, (x >> 18) << 5, 19)
    vc, vsc = enc(r, 5, x & 0x3FFFF, 18)
    vc = torch.where((r > 0) & (vsc > 0)[:, None], vc.clamp(min=1), vc)
    return p, mc | (m < 0).long() << 7, msc, vc, vsc


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_steps_in_8_bits_bit_for_bit(dtype, odd):
    sizes = SIZES * 6                                               # 78 tensors: two launches
    p, g, m, v, sm, sv, intact = _case(sizes, dtype, 8, 5, odd)
    decay = [WD * (i % 2) for i in range(len(sizes))]
    for i, x in enumerate(g):                                       # a wide range inside a block, whole blocks of zeros, tiny gradients
        x.mul_(torch.exp2(torch.arange(x.numel(), device="cuda") % 23 - 16.0).to(dtype))
        if i % 5 == 4:
            x.zero_()
        if i % 5 == 3 and dtype != torch.float16:
            x.mul_(1e-18)
    plan = AdamWPlan(p, m, v, sm, sv, weight_decay=decay)
    pad = lambda x, n: torch.nn.functional.pad(x, (0, -x.numel() % n)).view(-1, n)  # noqa: E731
    for t in range(1, 4):
        before = [(pad(p[i].float(), 256), pad(m[i].long(), 256), sm[i].clone(), pad(v[i].long(), 256), sv[i].clone()) for i in range(len(sizes))]
        norm = plan.step(g, step=t, lr=LR, betas=(B1, B2), eps=EPS, max_norm=0.5, seed=9)
        c = (torch.tensor(0.5, device="cuda") / (norm + 1e-6)).clamp(max=1.0)
        for i, n in enumerate(sizes):
            pb, mb, msb, vb, vsb = before[i]
            key = (i * 0x85157AF5 + 9 * 0x9E3779B1 + t * 0xC2B2AE3D) & 0xFFFFFFFF
            want = _mirror8(pb, pad(g[i].float(), 256), c, mb, msb, vb, vsb, t, decay[i], key)
            assert torch.equal(p[i], want[0].view(-1)[:n].to(dtype)), (t, n, "p")
            assert torch.equal(m[i].long(), want[1].view(-1)[:n]) and torch.equal(sm[i], want[2]), (t, n, "m")
            assert torch.equal(v[i].long(), want[3].view(-1)[:n]) and torch.equal(sv[i], want[4]), (t, n, "v")
            assert bool((adamw_moment(m[i], sm[i])[g[i] == 0].abs() <= 0).all()) or t > 1
    assert intact()


@pytest.mark.gpu
def test_8_bit_moments_follow_a_change_of_scale():
    """After half of every block's gradients shrink to 0.3, a second moment rounded to the nearest code would stay where it was; with
    probabilistic rounding the mean of log(sqrt(v) / sqrt(v in 64 bits)) over 32 768 elements goes to zero and its spread stays that of the
    rounding: per step one code step (<= 2^-5) is taken with probability d / step, a variance of d * step with d <= 0.0005 (b2 = 0.999) times
    a memory of 1 / (2 * 0.0005): spread <= sqrt(2^-5 / 2) = 0.125, mean within 0.125^2 of zero (Jensen) plus 0.125 / sqrt(32768)."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    n, b2 = 32768, 0.999
    p, m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda", dtype=torch.uint8), torch.zeros(n, device="cuda", dtype=torch.uint8)
    sm, sv = torch.zeros(n // 256, device="cuda"), torch.zeros(n // 256, device="cuda")
    plan = AdamWPlan([p], [m], [v], [sm], [sv])
    size = torch.exp(torch.randn(n, generator=gen, device="cuda"))
    size = size.clamp(max=8.0).clamp(min=0.5)                       # inside the format's normal range of the block's largest
    vd = torch.zeros(n, device="cuda", dtype=torch.float64)
    for t in range(1, 2401):
        g = size * (torch.randn(n, generator=gen, device="cuda"))
        if t > 400:
            g[::2] *= 0.3
        plan.step([g], step=t, lr=1e-4, betas=(0.9, b2))
        vd = b2 * vd + (1 - b2) * g.double().square()
    d = torch.log(adamw_moment(v, sv, squared=True).double().sqrt() / vd.sqrt())
    for part in (d[::2], d[1::2]):
        assert abs(float(part.mean())) <= 0.125 ** 2 + 0.125 / 128 and float(part.std()) <= 0.125, (float(part.mean()), float(part.std()))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite(bits):
    p, g, m, v, sm, sv, _ = _case([600], torch.float32, bits, 1)
    plan = AdamWPlan(p, m, v, sm, sv) if bits == 8 else AdamWPlan(p, m, v)
    before = p[0].clone()
    g[0][10], g[0][300] = float("nan"), float("inf")
    plan.step(g, step=1, lr=LR)
    assert bool(torch.isfinite(p[0][torch.arange(600, device="cuda") % 290 != 10]).all()) and bool(torch.isnan(p[0][10]))
    if bits == 8:                                                   # the scale of a block that holds one is NaN; the others go on
        assert torch.isnan(sm[0]).tolist() == [True, True, False] and torch.isnan(adamw_moment(m[0], sm[0])[:512]).all()
    else:
        assert bool(torch.isnan(m[0][10])) and bool(torch.isinf(m[0][300])) and bool(torch.isfinite(m[0][11:300]).all())
    p, g, m, v, sm, sv, _ = _case([600], torch.float32, bits, 1)
    plan = AdamWPlan(p, m, v, sm, sv) if bits == 8 else AdamWPlan(p, m, v)
    g[0][10] = float("nan")
    norm = plan.step(g, step=1, lr=LR, max_norm=1.0)                # a norm that is NaN makes every gradient NaN, as clip_grad_norm_ does
    assert bool(torch.isnan(norm)) and bool(torch.isnan(p[0]).all())
    assert torch.equal(before[:0], p[0][:0])


@pytest.mark.gpu
def test_norm_is_exact_for_large_and_small_values():
    g = [torch.full((100003,), 1e19, device="cuda"), torch.full((5,), 1e-25, device="cuda")]
    st = lambda: [torch.zeros_like(x) for x in g]  # noqa: E731
    plan = AdamWPlan(st(), st(), st())
    n = plan.step(g, step=1, lr=0.0, max_norm=math.inf)             # squares beyond fp32's range
    assert abs(float(n) - 1e19 * math.sqrt(100003)) <= 2 ** -23 * float(n)
    n = plan.step([torch.zeros_like(g[0]), g[1]], step=2, lr=0.0, max_norm=1.0)
    assert abs(float(n) - 1e-25 * math.sqrt(5)) <= 2 ** -23 * float(n)


@pytest.mark.gpu
def test_plan_refusals_on_the_device():
    z = lambda n, dt=torch.float32: torch.zeros(n, device="cuda", dtype=dt)  # noqa: E731
    p = z(300)
    with pytest.raises(_lib.NmrfHipError, match="twice"):
        AdamWPlan([p, p], [z(300), z(300)], [z(300), z(300)])
    with pytest.raises(_lib.NmrfHipError, match="contiguous"):
        AdamWPlan([z(600)[::2]], [z(300)], [z(300)])
    with pytest.raises(_lib.NmrfHipError, match="elements"):
        AdamWPlan([p], [z(299)], [z(300)])
    with pytest.raises(_lib.NmrfHipError, match="elements"):
        AdamWPlan([p], [z(300, torch.uint8)], [z(300, torch.uint8)], [z(1)], [z(2)])
    with pytest.raises(_lib.NmrfHipError, match="expected"):
        AdamWPlan([p], [z(300, torch.bfloat16)], [z(300)])
    plan = AdamWPlan([p], [z(300)], [z(300)])
    for bad, what in (([z(300, torch.bfloat16)], "expected"), ([z(299)], "elements"), ([z(600)[::2]], "contiguous"), ([torch.zeros(300)], "MI355X only")):
        with pytest.raises(_lib.NmrfHipError, match=what):
            plan.step(bad, step=1, lr=LR)
    with pytest.raises(ValueError, match="gradients"):
        plan.step([], step=1, lr=LR)
    with pytest.raises(ValueError, match="counts from 1"):
        plan.step([z(300)], step=0, lr=LR)
    p.data = z(300)
    with pytest.raises(_lib.NmrfHipError, match="new storage"):
        plan.step([z(300)], step=1, lr=LR)
    with pytest.raises(_lib.NmrfHipError, match="scales"):
        adamw_moment(z(300, torch.uint8), z(1))
    graph = torch.cuda.CUDAGraph()
    q = [z(300)]
    plan = AdamWPlan(q, [z(300)], [z(300)])
    g = [z(300)]
    with pytest.raises(_lib.NmrfHipError, match="captured"):
        with torch.cuda.graph(graph):
            plan.step(g, step=1, lr=LR)


@pytest.mark.gpu
def test_step_on_another_stream_and_version_counters():
    p, g, m, v, _, _, _ = _case([5000, 70001], torch.float32, 32, 7)
    q, h, m2, v2, _, _, _ = _case([5000, 70001], torch.float32, 32, 7)
    AdamWPlan(p, m, v).step(g, step=1, lr=LR, max_norm=0.1)
    plan, was = AdamWPlan(q, m2, v2), q[0]._version
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        plan.step(h, step=1, lr=LR, max_norm=0.1)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(p + m + v, q + m2 + v2))
    assert q[0]._version > was


# ---- the optimizer ------------------------------------------------------------------------------------------------------------------------
def _model(seed):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(37, 96), torch.nn.GELU(), torch.nn.LayerNorm(96), torch.nn.Linear(96, 64), torch.nn.Linear(64, 5)).cuda()


def _groups(m):
    vec = [p for p in m.parameters() if p.dim() == 1]
    return [{"params": [p for p in m.parameters() if p.dim() > 1], "lr": 2e-3}, {"params": vec, "lr": 1e-3, "weight_decay": 0.0}]


@pytest.mark.gpu
def test_optimizer_takes_torchs_steps():
    """Ten steps from the same gradients: every parameter within the sum over the steps of torch's and this step's roundings (9 of the update,
    3 of the parameter each, twice; moments: 12 roundings of each step's share, which sum to 12 of the moment)."""
    a, b = _model(1), _model(1)
    oa, ob = torch.optim.AdamW(_groups(a), weight_decay=0.05), O.AdamW(_groups(b), weight_decay=0.05)
    sched = [torch.optim.lr_scheduler.OneCycleLR(o, [2e-3, 1e-3], 40, pct_start=0.05, cycle_momentum=False) for o in (oa, ob)]
    gen = torch.Generator(device="cuda").manual_seed(2)
    pmax = [p.detach().abs() + 0.1 for p in a.parameters()]
    for t in range(10):
        for i, (p, q) in enumerate(zip(a.parameters(), b.parameters())):
            if t == 3 and i == 2:                                   # a step without a gradient: skipped, its own step count
                p.grad = q.grad = None
                continue
            p.grad = torch.randn(p.shape, generator=gen, device="cuda")
            q.grad = p.grad.clone()
        n = torch.nn.utils.clip_grad_norm_(a.parameters(), 1.0)
        oa.step()
        ob.step(max_norm=1.0)
        for s in sched:
            s.step()
        assert abs(float(n) - float(ob.grad_norm)) <= 2e-6 * float(n)
    for p, q, big in zip(a.parameters(), b.parameters(), pmax):
        # |update| <= lr * sqrt(t) bounded by 10 lr; 2 * 2^-24 * (3 |p| + 40 |update|) a step
        assert bool(((p - q).abs() <= 10 * 2 ** -23 * (3 * big + 40 * 2e-2)).all())
    sd = ob.state_dict()
    assert {k: float(s["step"]) for k, s in sd["state"].items()} == {k: float(s["step"]) for k, s in oa.state_dict()["state"].items()}
    c = _model(1)
    oc = torch.optim.AdamW(_groups(c), weight_decay=0.05)
    oc.load_state_dict(sd)
    assert torch.equal(oc.state[next(c.parameters())]["exp_avg"], ob.state[next(b.parameters())]["exp_avg"])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_train_step_on_the_model(bits):
    """train_step drives the optimizer of build_optimizer(..., state_bits): its first step from the same gradients is torch's (32 bits; 8 bits
    round the moments after they have been used) within the roundings of clip and step, and the kernels' packed weights follow the update."""
    from nmrf_amd.models.criterion import build_criterion
    from nmrf_amd.train import build_optimizer, train_step
    from tests.util import build_product, golden, golden_images, make_cfg
    import warnings
    g = golden("e2e_train")
    md = int(g["max_disp"])
    cfg = make_cfg(md)
    img1, img2 = golden_images(g)
    after = []
    for b in (None, bits):
        model = build_product(md, "cuda").train().enable_grad_slice()
        opt = build_optimizer(model, cfg, state_bits=b)
        was = {k: p.detach().clone() for k, p in model.named_parameters()}
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            losses = [train_step(model, build_criterion(cfg), opt, {"img1": img1, "img2": img2, "disp": torch.from_numpy(g["gt"]).clone(),
                                                                    "valid": torch.from_numpy(g["valid"])}, grad_clip=cfg.SOLVER.GRAD_CLIP)[0]
                      for _ in range(2)]
            if len(after) == 0 or b is not None:
                after.append((losses, was, {k: p.detach().clone() for k, p in model.named_parameters()}, opt))
    (la, wa, pa, _), (lb, wb, pb, opt) = after
    assert isinstance(opt, O.AdamW) and all(torch.equal(wa[k], wb[k]) for k in wa) and la[0] == lb[0]
    assert lb[1] != lb[0]                                           # the second forward ran on the updated weights
    lr = cfg.SOLVER.BASE_LR
    moved = 0
    # Two steps from moments of zero.  The first is lr long (m / bc1 = g, sqrt(v / bc2) = |g|), the second at most lr (0.9 * 0.1 |g1| / 0.19) /
    # sqrt(0.999 * 0.001 g1^2 / 0.001999) + lr (0.1 / 0.19) / sqrt(0.001 / 0.001999) = lr (0.67 + 0.75): 2.42 lr.  With 8-bit moments between
    # them the first share changes by the quotient of the two roundings: m goes up by less than a step and at most to twice its value or, below
    # one step, to one step 2^-10 s_m <= 2^-10 m_max; sqrt(v) goes down to no less than half or, below two steps, to one step 2^-11 s_v >
    # 2^-12 r_max: at most a factor of 4, 1 + 4 * 0.67 + 0.75 = 4.43 lr.
    longest = {None: 2.45, 32: 2.45, 8: 4.45}
    for k in pa:
        for p, b in ((pa[k], None), (pb[k], bits)):
            assert bool(((p - wa[k]).abs() <= longest[b] * lr * (1 + wa[k].abs())).all()), (k, b)
        moved += not torch.equal(pb[k], wa[k])
    assert moved == sum(not torch.equal(pa[k], wa[k]) for k in pa) > 200
    if bits == 8:
        assert any("exp_avg_scale" in s for s in opt.state.values())


@pytest.mark.gpu
def test_optimizer_in_8_bits_resumes_bit_for_bit(tmp_path):
    a, b = _model(1), _model(1)
    oa, ob = (O.AdamW(_groups(m), state_bits=8, min_8bit_size=1000, seed=5) for m in (a, b))
    gen = torch.Generator(device="cuda").manual_seed(2)
    grads = [[torch.randn(p.shape, generator=gen, device="cuda") for p in a.parameters()] for _ in range(6)]

    def run(m, o, gs):
        for g in gs:
            for p, x in zip(m.parameters(), g):
                p.grad = x.clone()
            o.step(max_norm=1.0)
    run(a, oa, grads)
    run(b, ob, grads[:3])
    torch.save({"o": ob.state_dict(), "m": b.state_dict()}, tmp_path / "c.pth")
    ck = torch.load(tmp_path / "c.pth", weights_only=True)
    c = _model(9)
    c.load_state_dict(ck["m"])
    oc = O.AdamW(_groups(c), state_bits=8, min_8bit_size=1000, seed=5)
    oc.load_state_dict(ck["o"])
    assert oc.state[next(c.parameters())]["exp_avg"].dtype == torch.uint8
    run(c, oc, grads[3:])
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), c.parameters()))
    w = next(c.parameters())
    m, v = oc.moments(w)
    assert m.shape == w.shape and m.dtype == torch.float32 and bool((v >= 0).all())
    small = [p for p in c.parameters() if p.numel() < 1000]
    assert all(oc.state[p]["exp_avg"].dtype == torch.float32 for p in small)


@pytest.mark.gpu
def test_optimizer_sees_new_storage_and_mixed_types():
    a = [torch.nn.Parameter(torch.ones(500, device="cuda")), torch.nn.Parameter(torch.ones(9000, device="cuda", dtype=torch.bfloat16))]
    o = O.AdamW(a, lr=0.1, weight_decay=0.0, state_bits=8)
    for _ in range(2):
        for p in a:
            p.grad = torch.ones_like(p)
        o.step(max_norm=1.0)
        a[0].data = a[0].data.clone()                               # e.g. a checkpoint load that rebinds the storage
    # constant gradients: m / sqrt(v) = 1 after the bias corrections, two steps of 0.1 (8 bits: codes within 2^-4 and 2^-5 of the moments)
    assert abs(float(a[0][0]) - 0.8) < 1e-5 and abs(float(a[1][0]) - 0.8) <= 0.1 * (2 ** -4 + 2 ** -5) * 1.5 + 0.8 * 2 ** -8
    assert abs(float(o.grad_norm) - math.sqrt(9500)) < 1e-3
    for b in (0.91, 0.92, 0.93):                                    # a schedule that moves the betas: no plan is kept for the old ones
        o.param_groups[0]["betas"] = (b, 0.999)
        o.step()
    assert len(o._plans) == 2
    o.state[a[0]]["step"] = o.state[a[1]]["step"] = 2
    a[0].grad = torch.ones(500, device="cuda")[:, None].expand(500, 1)[:, 0]
    a[1].grad = None
    o.step()
    assert o.state[a[1]]["step"] == 2 and o.state[a[0]]["step"] == 3


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_strided_gradients_of_several_types_step_as_contiguous_ones(bits):
    """The contiguous copies of strided gradients live until every type's update has been launched (a copy freed early is where the next
    type's copy, or the norm's partial sums, would go): the same bits as from contiguous gradients."""
    def run(strided):
        gen = torch.Generator("cpu").manual_seed(3)
        params = [torch.nn.Parameter(torch.randn(96, 128, generator=gen).to("cuda", t)) for t in (torch.float32, torch.bfloat16, torch.float16) * 2]
        o = O.AdamW(params, lr=0.01, state_bits=bits)
        for _ in range(3):
            for p in params:
                g = torch.randn(96, 128, generator=gen).to("cuda", p.dtype)
                p.grad = g.t().contiguous().t() if strided else g
            o.step(max_norm=0.5)
        return [p.detach() for p in params] + [o.grad_norm]

    assert run(True)[0].shape == (96, 128)
    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_plan_refuses_a_parameter_whose_layout_changed():
    p = torch.nn.Parameter(torch.ones(64, 128, device="cuda"))
    z = lambda: torch.zeros(64, 128, device="cuda")  # noqa: E731
    plan = AdamWPlan([p], [z()], [z()])
    plan.step([torch.ones(64, 128, device="cuda")], 1, 0.1)
    p.data = p.data.t()
    with pytest.raises(_lib.NmrfHipError, match="layout"):
        plan.step([torch.ones(128, 64, device="cuda")], 2, 0.1)
