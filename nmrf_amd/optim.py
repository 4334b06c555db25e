"""AdamW on the HIP kernels, with the moments in 32 or in 8 bits and the gradient clipping inside the step (the reference: torch.optim.AdamW
from build_optimizer, main.py:186-245, behind clip_grad_norm_, main.py:413-430).  nmrf_amd.train.build_optimizer(model, cfg, state_bits=...)
builds one with the reference's parameter groups; train_step and fit drive it."""
import operator

import numpy as np
import torch

from .ops.adamw import AdamWPlan, adamw_moment, clip_factor, refuse_capture


class AdamW(torch.optim.Optimizer):
    """AdamW(params, lr, betas, eps, weight_decay) with decoupled weight decay, on contiguous CUDA parameters in fp32, bf16 or fp16 (others raise).

    state_bits=32: state and checkpoints as torch.optim.AdamW's ({'step', 'exp_avg', 'exp_avg_sq'}): either loads the other's.
    state_bits=8: tensors of min_8bit_size elements or more hold their moments as uint8 codes with a fp32 scale for 256 elements (2.03 bytes a
    parameter instead of 8; {'step', 'exp_avg', 'exp_avg_scale', 'exp_avg_sq', 'exp_avg_sq_scale'}), smaller ones in 32 bits; seed: of the
    random bits of their rounding.

    step(max_norm=c) clips the global gradient norm on the way (torch.nn.utils.clip_grad_norm_'s factor, applied as the gradients are read:
    .grad itself is not rewritten) and leaves the norm in self.grad_norm, a 0-dim device tensor.  Parameters whose .grad is None are skipped,
    as in torch; a step whose set of parameters with gradients is another one than the last step's checks and lists them anew.  A step is not
    captured into a graph (it raises): lr and the step count are numbers of the host."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, min_8bit_size=4096, seed=0):
        if state_bits not in (32, 8):
            raise ValueError("AdamW: state_bits is 32 or 8, got %r" % (state_bits,))
        if not (lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0 and 0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("AdamW: lr %r, betas %r, eps %r, weight_decay %r" % (lr, betas, eps, weight_decay))
        self.state_bits, self.min_8bit_size, self.seed, self.grad_norm, self._plans = state_bits, int(min_8bit_size), int(seed), None, {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def _init_state(self, p):
        s = self.state[p]
        s["step"] = 0
        zeros = lambda n, dtype: torch.zeros(n, device=p.device, dtype=dtype)  # noqa: E731
        if self.state_bits == 8 and p.numel() >= self.min_8bit_size:
            blocks = -(-p.numel() // 256)
            s["exp_avg"], s["exp_avg_scale"] = zeros(p.shape, torch.uint8), zeros(blocks, torch.float32)
            s["exp_avg_sq"], s["exp_avg_sq_scale"] = zeros(p.shape, torch.uint8), zeros(blocks, torch.float32)
        else:
            s["exp_avg"], s["exp_avg_sq"] = zeros(p.shape, torch.float32), zeros(p.shape, torch.float32)
        return s

    def moments(self, p):
        """(first, second) moment of parameter p as fp32 tensors, whatever they are held in.  A parameter that has taken no step has none (KeyError)."""
        s = self.state.get(p)                                          # (a lookup by [p] would leave an empty entry behind)
        if not s:
            raise KeyError("AdamW: a parameter of shape %s has taken no step" % (tuple(p.shape),))
        if "exp_avg_scale" in s:
            return adamw_moment(s["exp_avg"], s["exp_avg_scale"]), adamw_moment(s["exp_avg_sq"], s["exp_avg_sq_scale"], squared=True)
        return s["exp_avg"], s["exp_avg_sq"]

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "min_8bit_size": self.min_8bit_size, "seed": self.seed}

    def __setstate__(self, state):
        super().__setstate__(state)
        self.grad_norm, self._plans = None, {}

    def _plan(self, key, items):
        """The plan of the parameters in items, kept while they and their state tensors are the same objects."""
        tensors = [t for p, s, _ in items for t in ((p, s["exp_avg"], s["exp_avg_sq"]) if key[2] == 32 else (
            p, s["exp_avg"], s["exp_avg_sq"], s["exp_avg_scale"], s["exp_avg_sq_scale"]))]
        had = self._plans.get(key)
        if had is not None and len(had[0]) == len(tensors) and all(map(operator.is_, had[0], tensors)) and had[1].unmoved():
            return had
        step = 3 if key[2] == 32 else 5
        return tensors, AdamWPlan(*(tensors[i::step] for i in range(step)))

    @torch.no_grad()
    def step(self, closure=None, max_norm=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if max_norm is not None and not max_norm > 0:
            raise ValueError("AdamW: max_norm %r is not positive" % (max_norm,))
        refuse_capture()
        sets = {}
        for group in self.param_groups:
            if group.get("amsgrad") or group.get("maximize"):
                raise NotImplementedError("AdamW: amsgrad and maximize are not supported")
            for p in group["params"]:
                if p.grad is not None:
                    s = self.state[p] if self.state.get(p) else self._init_state(p)
                    key = (p.device, p.dtype, 8 if "exp_avg_scale" in s else 32, tuple(group["betas"]))
                    sets.setdefault(key, []).append((p, s, group))
        self.grad_norm = None
        if not sets:
            return loss
        if len({k[0] for k in sets}) > 1 and max_norm is not None:
            raise NotImplementedError("AdamW: clipping over parameters on several devices")
        plans, held = [], []                                           # held: copies of strided gradients, until the update has been launched
        self._plans = {key: self._plan(key, items) for key, items in sets.items()}
        for key, items in sets.items():
            plan = self._plans[key][1]
            with torch.cuda.device(key[0]):
                grads = [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p, _, _ in items]
                plan.bind(grads)
            held.append(grads)
            plans.append((plan, key, items))
        coef = None
        if max_norm is not None:
            with torch.cuda.device(plans[0][0].device):
                self.grad_norm, coef = clip_factor([plan for plan, _, _ in plans], max_norm)
        for plan, key, items in plans:
            for _, s, _ in items:
                s["step"] += 1
            steps = [s["step"] for _, s, _ in items]
            groups = [g for _, _, g in items]
            same = groups[0] is groups[-1] and len(set(map(id, groups))) == 1
            pick = lambda k: groups[0][k] if same else [g[k] for g in groups]  # noqa: E731
            plan.decay = np.asarray(pick("weight_decay"), np.float64)
            with torch.cuda.device(key[0]):
                plan.update(steps[0] if len(set(steps)) == 1 else steps, pick("lr"), key[3], pick("eps"), coef, self.seed)
        return loss

    def state_dict(self):
        sd = super().state_dict()
        sd["state"] = {k: {**s, "step": torch.tensor(float(s["step"]))} for k, s in sd["state"].items() if s}
        return sd

    def load_state_dict(self, state_dict):
        """A checkpoint of this class (same state_bits for every tensor) or -- with 32-bit state -- of torch.optim.AdamW."""
        saved, own = state_dict["param_groups"], self.param_groups
        if [len(g["params"]) for g in saved] != [len(g["params"]) for g in own]:
            raise ValueError("loaded state dict has another set of parameter groups")
        new = {}
        for i, p in zip((i for g in saved for i in g["params"]), (p for g in own for p in g["params"])):
            s = state_dict["state"].get(i)
            if not s:
                continue
            eight = self.state_bits == 8 and p.numel() >= self.min_8bit_size
            if eight != ("exp_avg_scale" in s):
                raise ValueError("loaded state holds the moments of a %s tensor in %d bits, this optimizer in %d" % (
                    tuple(p.shape), 8 if "exp_avg_scale" in s else 32, 8 if eight else 32))
            if tuple(s["exp_avg"].shape) != tuple(p.shape):
                raise ValueError("loaded state is of a %s tensor, the parameter is %s" % (tuple(s["exp_avg"].shape), tuple(p.shape)))
            if s.get("max_exp_avg_sq") is not None:
                raise NotImplementedError("AdamW: amsgrad is not supported")
            codes = torch.uint8 if eight else torch.float32
            to = lambda k, dtype: s[k].detach().to(device=p.device, dtype=dtype, copy=True).contiguous()  # noqa: E731
            new[p] = {"step": int(s["step"]), "exp_avg": to("exp_avg", codes), "exp_avg_sq": to("exp_avg_sq", codes)}
            if eight:
                new[p].update(exp_avg_scale=to("exp_avg_scale", torch.float32), exp_avg_sq_scale=to("exp_avg_sq_scale", torch.float32))
        super().load_state_dict({"state": {}, "param_groups": saved})
        for group in self.param_groups:
            group["betas"] = tuple(group["betas"])
        self.state.update(new)
        self._plans = {}

