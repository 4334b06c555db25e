from .adamw import AdamWPlan, adamw_moment  # noqa: F401
from .blocks import gated_ffn, residual_norm  # noqa: F401
from .functions import MSDeformAttnFunction, ms_deform_attn_core_pytorch  # noqa: F401
from .modules import GatedFeedForward, MSDeformAttn, ResidualNorm  # noqa: F401
