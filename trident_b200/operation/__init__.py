from .attention import Attention
from .gated_residual_rms_norm import GatedResidualRMSNorm
from .geglu import GEGLU
from .layer_norm import LayerNorm
from .linear import Linear
from .masked_softmax import MaskedSoftmax
from .paged_attention import paged_attention, paged_cache_append
from .reduce import Mean, Sum, Var, VarMean
from .rms_norm import RMSNorm
from .rms_norm_geglu import RMSNormGEGLU
from .softmax import Softmax
from .window_attention import WindowAttention

__all__ = [
    "Attention", "GatedResidualRMSNorm", "GEGLU", "LayerNorm", "Linear", "MaskedSoftmax", "Mean", "RMSNorm",
    "RMSNormGEGLU", "Softmax", "Sum", "Var", "VarMean", "WindowAttention", "paged_attention", "paged_cache_append",
]
