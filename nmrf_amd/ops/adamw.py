"""One AdamW step over many tensors at once on the HIP kernels of csrc/adamw.hip (the reference steps torch.optim.AdamW behind
clip_grad_norm_, main.py:186-245, 413-430).  nmrf_amd.optim.AdamW is the optimizer on top of it."""
import math
import operator

import numpy as np
import torch

from .. import kernels as K
from .._lib import NmrfHipError

# (plain loops over hundreds of tensors cost more host time than the launches: whole-list passes in C)
_data_ptr, _numel, _get_device, _contiguous = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.is_contiguous
_dtype = operator.attrgetter("dtype")


def adamw_moment(code, scale, squared=False):
    """The fp32 values that 8-bit moments stand for (codes and scales of AdamWPlan / nmrf_amd.optim.AdamW); squared=True: the second moment."""
    return K.adamw_moment(code, scale, squared)


def refuse_capture():
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise NmrfHipError("an AdamW step is not captured into a graph: its step count and learning rate are numbers of the host, every replay "
                           "would repeat them")


def _addr(a):
    return a.__array_interface__["data"][0]


class AdamWPlan:
    """What a training program keeps for one list of parameters that step together: the checked tensors and the host tables the launch reads.

    params: CUDA tensors of one device and one type (fp32, bf16, fp16), contiguous, none that overlap.  exp_avgs, exp_avg_sqs: fp32 tensors of
    the same sizes, or uint8 ones with exp_avg_scales, exp_avg_sq_scales (fp32, one per started 256 elements): moments in 8 bits, zeros to
    begin with; no storage is shared.  weight_decay: one number, or one for each parameter.

        norm = plan.step(grads, step=t, lr=..., max_norm=1.0)

    updates parameters and moments in place: two launches for the gradient norm (max_norm=None: none) and one for every 84 (8-bit moments:
    56) tensors, on the current stream, with no read-back and no copy.  The plan holds the tensors; each step checks that the
    parameters' storage is where it was (the moments are the caller's to leave in place)."""

    def __init__(self, params, exp_avgs, exp_avg_sqs, exp_avg_scales=None, exp_avg_sq_scales=None, weight_decay=0.0):
        self.params, self.exp_avgs, self.exp_avg_sqs = list(params), list(exp_avgs), list(exp_avg_sqs)
        n = len(self.params)
        if n == 0:
            raise ValueError("AdamWPlan: no parameters")
        self.bits = 32 if exp_avg_scales is None else 8
        self.scales = [[], []] if self.bits == 32 else [list(exp_avg_scales), list(exp_avg_sq_scales or [])]
        self.device, self.dtype = self.params[0].device, self.params[0].dtype
        if self.dtype not in K.DTYPE_CODE:
            raise NmrfHipError("AdamWPlan: parameters are fp32, bf16 or fp16, got %s" % self.dtype)
        lists = [self.exp_avgs, self.exp_avg_sqs] + (self.scales if self.bits == 8 else [])
        if any(len(x) != n for x in lists):
            raise ValueError("AdamWPlan: %d parameters, but lists of %s" % (n, [len(x) for x in lists]))
        self.n = n
        self._numel = np.fromiter(map(_numel, self.params), np.int64, n)
        state = torch.float32 if self.bits == 32 else torch.uint8
        for tensors, dtype in ((self.params, self.dtype), (self.exp_avgs, state), (self.exp_avg_sqs, state)):
            self._check(tensors, dtype, self._numel)
        for tensors in self.scales[:2] if self.bits == 8 else ():
            self._check(tensors, torch.float32, -(-self._numel // K.ADAMW_BLOCK))
        decay = np.asarray(weight_decay, np.float64)
        if decay.shape not in ((), (n,)):
            raise ValueError("AdamWPlan: weight_decay is one number or one for each of the %d parameters" % n)
        self.decay = decay
        self.parts = int(np.sum(-(-self._numel // K.GRAD_SQSUM_CHUNK)))
        self._lists = [self.params, self.exp_avgs, self.exp_avg_sqs] + (self.scales if self.bits == 8 else [])
        self._tables = [np.fromiter(map(_data_ptr, x), np.uint64, n) for x in self._lists]
        if len(set(self._tables[0][self._numel > 0].tolist())) != int(np.sum(self._numel > 0)):
            raise NmrfHipError("AdamWPlan: a parameter is in the list twice")
        # (each tensor is updated in place by blocks of its own: none may reach into another)
        start = np.concatenate(self._tables)
        size = np.concatenate([np.fromiter(map(_numel, x), np.uint64, n) * np.uint64(x[0].element_size()) for x in self._lists])
        order = np.argsort(start[size > 0], kind="stable")
        start, end = start[size > 0][order], (start + size)[size > 0][order]
        if bool((end[:-1] > start[1:]).any()):
            raise NmrfHipError("AdamWPlan: parameters or moments share storage")
        # (a parameter's address is checked each step; the moments' storage is held, whatever becomes of the tensors)
        self._held = [list(map(torch.Tensor.detach, x)) for x in self._lists[1:]]
        self._g = np.zeros(n, np.uint64)
        self._hyper = np.zeros((n, 4), np.float32)
        self._betas = np.zeros(4, np.float32)
        self._order = np.arange(n, dtype=np.uint64) * np.uint64(0x85157AF5)
        self._key = np.zeros(n, np.uint32)

    def _check(self, tensors, dtype, sizes):
        if (set(map(_dtype, tensors)) == {dtype} and set(map(_get_device, tensors)) == {self.device.index} and all(map(_contiguous, tensors))
                and np.array_equal(np.fromiter(map(_numel, tensors), np.int64, self.n), sizes)):
            return
        for t, n in zip(tensors, sizes):                               # something is wrong: say what
            if not t.is_cuda:
                raise NmrfHipError("AdamW runs on the MI355X only: got a %s tensor (no CPU fallback exists by design)" % t.device)
            if t.device != self.device:
                raise NmrfHipError("tensors of one AdamW step live on different devices: %s and %s" % (self.device, t.device))
            if t.dtype != dtype:
                raise NmrfHipError("AdamW: expected %s, got %s" % (dtype, t.dtype))
            if t.layout is not torch.strided or not t.is_contiguous():
                raise NmrfHipError("AdamW: tensor must be contiguous")
            if t.numel() != n:
                raise NmrfHipError("AdamW: a tensor has %d elements, its parameter needs %d" % (t.numel(), n))

    def unmoved(self):
        """Whether every parameter still has the storage the tables name, and its layout (p.data = ... gives it another)."""
        return np.array_equal(np.fromiter(map(_data_ptr, self.params), np.uint64, self.n), self._tables[0]) and all(map(_contiguous, self.params))

    def bind(self, grads):
        """Check one step's gradients (parameter order, the parameters' type and sizes) and take their addresses: the caller keeps them until
        the update has been launched."""
        if len(grads) != self.n:
            raise ValueError("AdamWPlan: %d gradients for %d parameters" % (len(grads), self.n))
        self._check(grads, self.dtype, self._numel)
        self._g[:] = np.fromiter(map(_data_ptr, grads), np.uint64, self.n)
        refuse_capture()

    def sqsum(self, parts):
        """Partial sums of squares of the bound gradients into parts (fp64, self.parts entries)."""
        if parts.numel():
            K.grad_sqsum(self.n, _addr(self._g), _addr(self._numel), self.dtype, parts)

    def update(self, step, lr, betas, eps, grad_scale=None, seed=0):
        """The update from the bound gradients; step, lr, eps: numbers, or one for each parameter."""
        b1, b2 = float(betas[0]), float(betas[1])
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError("AdamW: betas %r are not in [0, 1)" % (betas,))
        one = not np.ndim(step)
        t = int(step) if one else np.asarray(step, np.float64)
        if (t < 1) if one else (t.shape != (self.n,) or t.min() < 1):
            raise ValueError("AdamW: step counts from 1")
        lr = np.asarray(lr, np.float64) if np.ndim(lr) else float(lr)
        h = self._hyper
        h[:, 0] = 1.0 - lr * self.decay
        h[:, 1] = lr / (1.0 - b1 ** t)
        h[:, 2] = 1.0 / (math.sqrt(1.0 - b2 ** t) if one else np.sqrt(1.0 - b2 ** t))
        h[:, 3] = eps
        self._betas[:] = (b1, 1.0 - b1, b2, 1.0 - b2)
        scales, key = (None, None), None
        if self.bits == 8:
            word = (int(seed) * 0x9E3779B1 & 0xFFFFFFFF) if one else 0
            t = np.uint64((word + t * 0xC2B2AE3D) & 0xFFFFFFFF) if one else (
                np.uint64(int(seed) * 0x9E3779B1 & 0xFFFFFFFF) + t.astype(np.uint64) * np.uint64(0xC2B2AE3D))
            self._key[:] = (self._order + t) & np.uint64(0xFFFFFFFF)
            scales, key = (_addr(self._tables[3]), _addr(self._tables[4])), _addr(self._key)
        p, m, v = (_addr(x) for x in self._tables[:3])
        K.adamw_step(self.n, p, _addr(self._g), m, v, scales[0], scales[1], _addr(self._numel), _addr(h), key, _addr(self._betas), self.dtype,
                     self.bits, grad_scale)
        torch.autograd.graph.increment_version(self.params)            # in place: autograd and the caches of packed weights go by the version

    @torch.no_grad()
    def step(self, grads, step, lr, betas=(0.9, 0.999), eps=1e-8, max_norm=None, seed=0):
        """One step; -> the gradients' total norm (0-dim device tensor) when max_norm is given, else None.  seed: of the random bits that round
        8-bit moments (with the step count and the tensor's place they are a function of it: the same calls give the same bits)."""
        if max_norm is not None and not max_norm > 0:
            raise ValueError("AdamW: max_norm %r is not positive" % (max_norm,))
        if self.device.index != torch.cuda.current_device():
            with torch.cuda.device(self.device):
                return self.step(grads, step, lr, betas, eps, max_norm, seed)
        if not self.unmoved():
            raise NmrfHipError("AdamWPlan: a parameter has new storage or another layout: build a new plan")
        self.bind(grads)
        norm = coef = None
        if max_norm is not None:
            norm, coef = clip_factor([self], max_norm)
        self.update(step, lr, betas, eps, coef, seed)
        return norm


def clip_factor(plans, max_norm):
    """(norm, factor) of clip_grad_norm_ over the bound gradients of several plans on the current device."""
    total = sum(p.parts for p in plans)
    parts = torch.empty(total, device=plans[0].device, dtype=torch.float64) if total else torch.zeros(1, device=plans[0].device, dtype=torch.float64)
    at = 0
    for p in plans:
        p.sqsum(parts[at:at + p.parts])
        at += p.parts
    return K.grad_norm_factor(parts, max_norm)
