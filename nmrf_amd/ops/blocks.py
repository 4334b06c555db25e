"""Operators of a training block as autograd Functions over the HIP kernels: the gated feed-forward block (csrc/gated_ffn.hip) and the norms
around a block with its gate and residual scale (csrc/residual_norm.hip).  They stand beside the reference's feed-forward, fc2(gelu(fc1 x))
(nmrf/models/NMP.py:337, 537, 675), its block tails, x + proj(attn) / x + mlp(norm2(x)) (NMP.py:337-364), their post-norm form
(NMP.py:366-382) and stochastic depth (nmrf/models/swin.py:228-233, 300-301)."""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import kernels as K
from .._lib import NmrfHipError

_PROXY = torch._C._TorchDispatchModeKey.PROXY
_GATE_ACTS = {None: 0, "sigmoid": 1, "tanh": 2}


def check_rows(name, names, tensors):
    """One device, one type of fp32 / bf16 / fp16, on the GPU; and no recording by operations (make_fx), which goes inside a Function and would hold
    nothing of the kernels but the allocation of their outputs."""
    if torch._C._len_torch_dispatch_stack() and torch._C._get_dispatch_mode(_PROXY) is not None:
        raise NmrfHipError("%s is not recorded by make_fx (torch.jit.trace holds it as one call)" % name)
    ref = tensors[0]
    dtype, device = ref.dtype, ref.device
    if not ref.is_cuda:
        raise NmrfHipError("%s runs on the MI355X only: %s is a %s tensor (no CPU fallback exists by design)" % (name, names[0], device))
    if dtype not in K.DTYPE_CODE:
        raise NmrfHipError("%s: %s is fp32, bf16 or fp16, got %s" % (name, names[0], dtype))
    for k, t in zip(names, tensors):
        if t is None or t is ref:
            continue
        if t.device != device:
            raise NmrfHipError("%s: tensors live on different devices: %s and %s" % (name, device, t.device))
        if t.dtype != dtype:
            raise NmrfHipError("%s: %s is %s, expected %s" % (name, k, t.dtype, dtype))


def refuse_captured_backward(name):
    """A captured backward pass that accumulates into leaves does so on the stream their first graph was built on; with an eager graph of the same
    leaves alive that is another stream, and the capture takes the process down.  Whether a pass goes on to leaves or returns its gradients
    (torch.autograd.grad) cannot be seen from a node of it: all are refused.  Forward passes are captured freely."""
    if torch.cuda.is_current_stream_capturing():
        raise NmrfHipError("%s: a backward pass is not captured into a graph (capture the forward pass, or run it eagerly)" % name)


def differentiated(*tensors):
    """Whether a call goes through its Function.  A backward pass may follow (a Function does not see that gradients are switched off); or a
    forward-mode derivative is being taken, which the kernels alone would drop and the Function refuses; or a trace is being recorded, which
    holds a Function as one node and of the kernels alone nothing but the allocation of their outputs."""
    if torch.is_grad_enabled():
        for t in tensors:                                           # (a generator expression costs half a microsecond more)
            if t is not None and t.requires_grad:
                return True
    return forward_ad._current_level >= 0 or torch._C._is_tracing()


class ResidualNormFn(torch.autograd.Function):
    # (checks and layout belong to the forward pass: a recorded trace calls it again, with tensors of other sizes)
    @staticmethod
    def forward(ctx, *call):
        args, spec = _norm_call(*call)
        ctx.save_for_backward(*args)
        ctx.spec = spec
        ctx.set_materialize_grads(False)
        out, h = K.residual_norm(*args, spec)
        return (out, h) if spec.next else out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_h=None):
        refuse_captured_backward("residual_norm")
        saved = ctx.saved_tensors
        if d_out is None and d_h is None:
            return (None,) * 9
        d_out, d_h = (None if d is None else d.contiguous() for d in (d_out, d_h))
        want = [n and t is not None for n, t in zip(ctx.needs_input_grad[2:8], saved[2:])]
        return (*K.residual_norm_backward(*saved, d_out, d_h, ctx.spec, want), None)


# (while a trace is being recorded, sizes are tensors: int() where one is kept)
def _gate_layout(x, gate):
    """(rows that share a gate row, 1 or C) of a gate of shape `gate` that broadcasts over shape `x` from some dimension on."""
    shape = (1,) * (len(x) - len(gate)) + gate
    lead, c = x[:-1], x[-1]
    keep = next((k for k in range(len(lead) + 1) if shape[:k] == lead[:k] and all(n == 1 for n in shape[k:-1])), None)
    if len(gate) > len(x) or len(gate) < 1 or shape[-1] not in (1, c) or keep is None:
        raise ValueError("residual_norm: a gate of shape %s does not share one row with whole trailing dimensions of %s: its leading dimensions "
                         "are x's up to some point and 1 behind it, its last one %d or 1" % (tuple(gate), tuple(x), c))
    rows = 1
    for n in lead[keep:]:
        rows *= int(n)
    return max(rows, 1), int(shape[-1])


def _norm_call(x, y, gate, vec, post_w, post_b, next_w, next_b, options):
    """residual_norm's arguments checked: the contiguous tensors, and the call's numbers."""
    kind, gate_act, scale_value, post, nxt, eps = options
    shape = x.shape
    if shape != y.shape or not shape:
        raise ValueError("residual_norm: x %s and y %s differ" % (tuple(shape), tuple(y.shape)))
    c = int(shape[-1])
    if not 1 <= c <= 8192:
        raise ValueError("residual_norm: %d channels are not in 1 ... 8192" % c)
    check_rows("residual_norm", ("x", "y", "gate"), (x, y, gate))
    device, of = x.device, None                                         # of: the parameters' type
    params = (vec, post_w, post_b, next_w, next_b)
    for k, t in zip(("scale", "post_weight", "post_bias", "next_weight", "next_bias"), params):
        if t is None:
            continue
        if t.shape != (c,):
            raise ValueError("residual_norm: %s has shape %s, expected (%d,)" % (k, tuple(t.shape), c))
        if t.device != device or not t.is_contiguous():
            raise NmrfHipError("residual_norm: %s is not a contiguous tensor on %s" % (k, device))
        if of is None:
            of = t.dtype
        if t.dtype != of or (of != x.dtype and of != torch.float32):
            raise NmrfHipError("residual_norm: weights, biases and the scale vector are all %s or all torch.float32, got %s for %s" % (x.dtype, t.dtype, k))
    rows, cols = (1, 1) if gate is None else _gate_layout(shape, gate.shape)
    spec = K.ResidualNormSpec(int(x.numel()) // c, c, kind, eps, rows, cols, gate_act, scale_value, post, nxt, int(of == torch.float32), K.DTYPE_CODE[x.dtype])
    return (x.contiguous(), y.contiguous(), None if gate is None else gate.contiguous(), *params), spec


def residual_norm(x, y, next_norm=None, post_norm=None, gate=None, gate_act=None, scale=None, kind="layer", eps=1e-5):
    """out = x + scale * act(gate) * z with z = norm(y) (post_norm) or y, and h = norm(out) for the next block (next_norm): the norms before and
    after a block, its gate and its residual scale in one pass.  -> (out, h), or out alone without next_norm.

    x, y: [..., C], C <= 8192, fp32 / bf16 / fp16 (copied if not contiguous).  post_norm, next_norm: (weight, bias) of the norm, either of them
    may be None; kind "layer" or "rms".  gate: broadcasts over x with x's leading dimensions up to some point and 1 behind it -- [..., C] per
    element, [..., 1] per row, [B, 1, C] or [B, 1, 1] per sample (conditioned blocks, stochastic depth: zeros and 1 / keep) --, through
    gate_act None, "sigmoid" or "tanh".  scale: a number, or a vector over the channels.  Weights, biases and the scale vector are all in x's
    type or all in fp32.  Differentiable in every tensor, once and backwards (forward mode raises); statistics and sums in fp32, the same bits
    every run.  The forward pass may be captured into a graph or recorded by torch.jit.trace, the backward pass may not be captured (it raises)."""
    if kind not in ("layer", "rms"):
        raise ValueError("residual_norm: kind is 'layer' or 'rms', got %r" % (kind,))
    if gate_act not in _GATE_ACTS:
        raise ValueError("residual_norm: gate_act is None, 'sigmoid' or 'tanh', got %r" % (gate_act,))
    if not eps >= 0:
        raise ValueError("residual_norm: eps %r" % (eps,))
    post_w, post_b = post_norm if post_norm is not None else (None, None)
    next_w, next_b = next_norm if next_norm is not None else (None, None)
    vec = scale if isinstance(scale, torch.Tensor) else None
    tensors = (x, y, gate, vec, post_w, post_b, next_w, next_b)
    options = (int(kind == "rms"), _GATE_ACTS[gate_act], 1.0 if scale is None or vec is not None else float(scale), int(post_norm is not None),
               int(next_norm is not None), float(eps))
    if differentiated(*tensors):
        return ResidualNormFn.apply(*tensors, options)
    args, spec = _norm_call(*tensors, options)
    out, h = K.residual_norm(*args, spec)
    return (out, h) if spec.next else out


_FFN_ACTS = {"silu": 0, "gelu": 1, "relu": 2}
_FFN_NAMES = ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")


class GatedFfnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *call):
        args = _ffn_call(*call[:7])
        ctx.act, ctx.shape = _FFN_ACTS[call[7]], call[0].shape
        y, h, g, u, amax = K.gated_ffn(*args, ctx.act, any(ctx.needs_input_grad))
        ctx.save_for_backward(*args[:4], h, g, u, amax)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        refuse_captured_backward("gated_ffn")
        dx, *rest = K.gated_ffn_backward(*ctx.saved_tensors, dy.contiguous(), ctx.act, ctx.needs_input_grad[:7])
        return (None if dx is None else dx.view(ctx.shape), *rest, None)


def _ffn_call(x, w_gate, w_up, w_down, b_gate, b_up, b_down):
    """gated_ffn's tensors checked: contiguous, x as rows."""
    if x.dim() < 1 or w_gate.dim() != 2 or w_down.dim() != 2:
        raise ValueError("gated_ffn: x [..., D], w_gate, w_up [F, D], w_down [D', F]; got %s, %s, %s" % (
            tuple(x.shape), tuple(w_gate.shape), tuple(w_down.shape)))
    d, f, do = int(x.shape[-1]), int(w_gate.shape[0]), int(w_down.shape[0])
    for name, t, want in zip(_FFN_NAMES[1:], (w_gate, w_up, w_down, b_gate, b_up, b_down), ((f, d), (f, d), (do, f), (f,), (f,), (do,))):
        if t is not None and t.shape != want:
            raise ValueError("gated_ffn: %s has shape %s, expected %s" % (name, tuple(t.shape), want))
    if min(d, f, do) < 1 or max(d, f, do) > 1 << 22:
        raise ValueError("gated_ffn: widths %d, %d, %d are not in 1 ... 2^22" % (d, f, do))
    check_rows("gated_ffn", _FFN_NAMES, (x, w_gate, w_up, w_down, b_gate, b_up, b_down))
    rows = int(x.numel()) // d
    if rows > 0x7fffffff - 256:
        raise ValueError("gated_ffn: %d rows" % rows)
    return [None if t is None else t.contiguous() for t in (x.reshape(rows, d), w_gate, w_up, w_down, b_gate, b_up, b_down)]


def gated_ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, act="silu"):
    """y = (act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down: both projections, the activation and the product in one kernel, the
    second matrix in another.

    x: [..., D]; w_gate, w_up: [F, D]; w_down: [D', F]; biases [F], [F], [D'], each may be None; one type, fp32 / bf16 / fp16 (copied where not
    contiguous; autocast does not cast here).  act: "silu", "gelu" (erf; zero below -7) or "relu".  16-bit types multiply on the matrix pipe as
    they are, sums in fp32; h and the gradients of both projections are rounded to the type on the way, as operands of the next product, the
    projections are kept in fp32 for the backward pass.  fp32 is multiplied as scaled fp16 pairs: errors of 2^-22 of a value and 2^-38 of the largest
    entry that shares its scale (w_gate with w_up, the gradients of both projections), and an infinite input gives NaN.  Differentiable in every
    tensor, once and backwards (forward mode raises), the same bits every run.  Up to 64 rows without gradients (decoding) stream the weights
    once.  The forward pass may be captured into a graph or recorded by torch.jit.trace, the backward pass may not be captured (it raises)."""
    if act not in _FFN_ACTS:
        raise ValueError("gated_ffn: act is 'silu', 'gelu' or 'relu', got %r" % (act,))
    tensors = (x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    y = GatedFfnFn.apply(*tensors, act) if differentiated(*tensors) else K.gated_ffn(*_ffn_call(*tensors), _FFN_ACTS[act], False)[0]
    return y.view(*x.shape[:-1], y.shape[-1])
