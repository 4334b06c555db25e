"""residual_norm and gated_ffn under forward-mode differentiation and torch.jit.trace, with gradients off or on.  On the CPU the two forward kernels are replaced
by ones that write through the outputs' addresses, as the library does (nothing that torch could differentiate or record); `plain` is what they
compute there.  On the GPU the calls are the library's."""
import contextlib
import ctypes

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from nmrf_amd import _lib
from nmrf_amd.ops import blocks

pytestmark = pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")


def put(out, value):
    value = value.detach().contiguous()
    assert out.shape == value.shape
    ctypes.memmove(out.data_ptr(), value.data_ptr(), value.numel() * 4)


def plain_norm(x, y, w):
    return x + y, (x + y) * w


def plain_ffn(x, wg, wu, wd):
    return (torch.relu(x @ wg.t()) * (x @ wu.t())) @ wd.t()


@pytest.fixture
def by_address(monkeypatch):
    def norm(x, y, gate, scale, post_w, post_b, next_w, next_b, s):
        assert s.t == x.numel() // x.shape[-1] and s.c == x.shape[-1] and all(type(n) in (int, float) for n in s) and (gate is None or gate.numel() * s.gate_rows == s.t)
        out, h = torch.empty_like(x), torch.empty_like(x)
        with torch.no_grad():
            f = 1.0 if gate is None else gate.view(-1, 1).repeat_interleave(s.gate_rows, 0).view(*x.shape[:-1], 1)
            want = plain_norm(x, y * f, next_w)
            put(out, want[0])
            put(h, want[1])
        return out, h

    def ffn(x, wg, wu, wd, bg, bu, bd, act, keep):
        y = torch.empty(x.shape[0], wd.shape[0])
        with torch.no_grad():
            put(y, plain_ffn(x, wg, wu, wd))
        return y, *(torch.zeros(x.shape[0], wg.shape[0]) for _ in range(3)), None
    monkeypatch.setattr(blocks.K, "residual_norm", norm)
    monkeypatch.setattr(blocks.K, "gated_ffn", ffn)
    monkeypatch.setattr(blocks, "check_rows", lambda *a: None)
    monkeypatch.setattr(blocks, "refuse_captured_backward", lambda name: None)


def calls(device, rows=6, leaf=False):
    gen = torch.Generator().manual_seed(rows)
    r = lambda *s: torch.randn(s, generator=gen).to(device).requires_grad_(leaf)  # noqa: E731
    gen_w = torch.Generator().manual_seed(99)
    w = [torch.randn(s, generator=gen_w).to(device) for s in ((8,), (16, 8), (16, 8), (24, 16))]
    return ((lambda x, y, g: blocks.residual_norm(x, y, (w[0], None), gate=g), (r(2, rows, 8), r(2, rows, 8), r(2, 1, 1))),
            (lambda x: blocks.gated_ffn(x, *w[1:], act="relu"), (r(2, rows, 8),)))


def outputs(o):
    return o if isinstance(o, tuple) else (o,)


def tangents_are_refused(device):
    for f, args in calls(device):
        for off in (contextlib.nullcontext, torch.no_grad):
            with forward_ad.dual_level(), off():
                for i in range(len(args)):
                    dual = [forward_ad.make_dual(a, torch.ones_like(a)) if i == k else a for k, a in enumerate(args)]
                    with pytest.raises(NotImplementedError, match="jvp"):
                        f(*dual)
                inside = outputs(f(*args))                          # without a tangent: the values as ever
            assert all(torch.equal(a, b) for a, b in zip(inside, outputs(f(*args))))


def traces_compute(device):
    for leaf in (False, True):
        with contextlib.nullcontext() if leaf else torch.no_grad():
            for (f, args), (_, other) in zip(calls(device, leaf=leaf), calls(device, rows=11, leaf=leaf)):
                traced = torch.jit.trace(f, args, check_trace=False)
                for a in (args, other):                             # (the second time with another number of rows)
                    torch.full((1 << 16,), 3.0, device=device)      # what fresh memory may hold
                    for got, want in zip(outputs(traced(*a)), outputs(f(*a))):
                        assert torch.equal(got, want) and got.requires_grad == want.requires_grad == leaf
    (f, (x, y, g)), _ = calls(device)
    with torch.no_grad():
        traced = torch.jit.trace(f, (x, y, g), check_trace=False)
        with pytest.raises(Exception, match="differ"):              # sizes are checked again where a trace is run
            traced(x, y[:, :3], g)


def test_forward_mode_is_refused(by_address):
    tangents_are_refused("cpu")


def test_traced_calls_compute(by_address):
    traces_compute("cpu")


def test_outputs_may_be_changed_in_place(by_address):
    for f, args in calls("cpu", leaf=True):
        for o in outputs(f(*args)):
            o += 1.0
            assert o.requires_grad


def recordings_are_refused(device):
    for leaf in (False, True):
        for f, args in calls(device, leaf=leaf):
            with pytest.raises(_lib.NmrfHipError, match="make_fx"):
                make_fx(f)(*args)


def test_recording_by_operations_is_refused():
    recordings_are_refused("cpu")


@pytest.mark.gpu
def test_recording_by_operations_is_refused_on_the_device():
    recordings_are_refused("cuda")


@pytest.mark.gpu
def test_forward_mode_is_refused_on_the_device():
    tangents_are_refused("cuda")


@pytest.mark.gpu
def test_traced_calls_compute_on_the_device():
    traces_compute("cuda")
