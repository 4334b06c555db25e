"""`ops.modules.MSDeformAttn` (ops/modules/ms_deform_attn.py:28-130) on the HIP operator, and the modules of a training block on theirs."""
import math

import torch
import torch.nn.functional as F
from torch import nn

from .blocks import gated_ffn, residual_norm
from .functions import MSDeformAttnFunction


class MSDeformAttn(nn.Module):
    """Multi-scale deformable attention.  Parameters: sampling_offsets, attention_weights, value_proj, output_proj."""

    def __init__(self, d_model=256, n_levels=4, n_heads=8, n_points=4, ratio=1.0):
        super().__init__()
        if d_model % n_heads != 0:
            raise ValueError("d_model must be divisible by n_heads, but got {} and {}".format(d_model, n_heads))
        self.im2col_step = 64
        self.d_model, self.n_levels, self.n_heads, self.n_points, self.ratio = d_model, n_levels, n_heads, n_points, ratio
        self.sampling_offsets = nn.Linear(d_model, n_heads * n_levels * n_points * 2)
        self.attention_weights = nn.Linear(d_model, n_heads * n_levels * n_points)
        self.value_proj = nn.Linear(d_model, int(d_model * ratio))
        self.output_proj = nn.Linear(int(d_model * ratio), d_model)
        self._reset_parameters()

    def _reset_parameters(self):
        nn.init.zeros_(self.sampling_offsets.weight)
        ang = torch.arange(self.n_heads, dtype=torch.float32) * (2.0 * math.pi / self.n_heads)
        ring = torch.stack((ang.cos(), ang.sin()), -1)
        ring = ring / ring.abs().max(-1, keepdim=True)[0]
        ring = ring.view(self.n_heads, 1, 1, 2).repeat(1, self.n_levels, self.n_points, 1)
        ring = ring * torch.arange(1, self.n_points + 1, dtype=torch.float32).view(1, 1, -1, 1)
        with torch.no_grad():
            self.sampling_offsets.bias.copy_(ring.reshape(-1))
        nn.init.zeros_(self.attention_weights.weight)
        nn.init.zeros_(self.attention_weights.bias)
        nn.init.xavier_uniform_(self.value_proj.weight)
        nn.init.zeros_(self.value_proj.bias)
        nn.init.xavier_uniform_(self.output_proj.weight)
        nn.init.zeros_(self.output_proj.bias)

    def forward(self, query, reference_points, input_flatten, input_spatial_shapes, input_level_start_index,
                input_padding_mask=None):
        n, len_q, _ = query.shape
        _, len_in, _ = input_flatten.shape
        if not (input_flatten.is_cuda and torch.cuda.is_current_stream_capturing()):
            # (reads the device tensor back: the reference's check, ms_deform_attn.py:97; skipped while a hipGraph is being captured)
            assert int((input_spatial_shapes[:, 0] * input_spatial_shapes[:, 1]).sum()) == len_in
        value = self.value_proj(input_flatten)
        if input_padding_mask is not None:
            value = value.masked_fill(input_padding_mask[..., None], 0.0)
        value = value.view(n, len_in, self.n_heads, int(self.ratio * self.d_model) // self.n_heads)
        off = self.sampling_offsets(query).view(n, len_q, self.n_heads, self.n_levels, self.n_points, 2)
        aw = F.softmax(self.attention_weights(query).view(n, len_q, self.n_heads, self.n_levels * self.n_points), -1)
        aw = aw.view(n, len_q, self.n_heads, self.n_levels, self.n_points)
        if reference_points.shape[-1] == 2:
            norm = torch.stack((input_spatial_shapes[..., 1], input_spatial_shapes[..., 0]), -1)
            loc = reference_points[:, :, None, :, None, :] + off / norm[None, None, None, :, None, :]
        elif reference_points.shape[-1] == 4:
            loc = reference_points[:, :, None, :, None, :2] + off / self.n_points * reference_points[:, :, None, :, None, 2:] * 0.5
        else:
            raise ValueError("Last dim of reference_points must be 2 or 4, but get {} instead.".format(reference_points.shape[-1]))
        out = MSDeformAttnFunction.apply(value.contiguous(), input_spatial_shapes, input_level_start_index,
                                         loc.contiguous(), aw.contiguous(), self.im2col_step)
        return self.output_proj(out)


class GatedFeedForward(nn.Module):
    """y = down(act(gate(x)) * up(x)) on nmrf_amd.ops.gated_ffn: the gated form of the reference's Mlp (fc2(gelu(fc1 x)), nmrf/models/NMP.py:337, 537,
    675).  Parameters: gate, up [hidden, dim], down [out, hidden] (nn.Linear's layout and initialisation)."""

    def __init__(self, dim, hidden, out=None, act="silu", bias=True):
        super().__init__()
        self.act = act
        self.gate, self.up, self.down = nn.Linear(dim, hidden, bias), nn.Linear(dim, hidden, bias), nn.Linear(hidden, out or dim, bias)

    def forward(self, x):
        return gated_ffn(x, self.gate.weight, self.up.weight, self.down.weight, self.gate.bias, self.up.bias, self.down.bias, self.act)


class ResidualNorm(nn.Module):
    """(x, y) -> (out, h) on nmrf_amd.ops.residual_norm: out = x + scale * act(gate) * [post](y), h = next(out) -- the tail of a block and the norm in
    front of the next one (nmrf/models/NMP.py:337-364).  post: normalise the branch too.  layer_scale: a learned scale for each channel that
    begins at this value (None: none).  A gate is given with the call."""

    def __init__(self, dim, kind="layer", post=False, layer_scale=None, eps=1e-5, gate_act=None):
        super().__init__()
        self.kind, self.eps, self.gate_act, self.post = kind, eps, gate_act, post
        one = lambda v: nn.Parameter(torch.full((dim,), float(v)))  # noqa: E731
        self.weight, self.bias = one(1), (one(0) if kind == "layer" else None)
        if post:
            self.post_weight, self.post_bias = one(1), (one(0) if kind == "layer" else None)
        self.layer_scale = None if layer_scale is None else one(layer_scale)

    def forward(self, x, y, gate=None):
        return residual_norm(x, y, (self.weight, self.bias), (self.post_weight, self.post_bias) if self.post else None, gate, self.gate_act,
                             self.layer_scale, self.kind, self.eps)
