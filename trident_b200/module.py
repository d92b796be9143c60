"""nn.Module front ends (constructor arguments, parameter names, initialisation and
`extra_repr` follow trident/module.py so that state_dicts and printed models carry over).
"""

import math
from typing import Tuple, Union

import torch

from trident_b200 import function, util

__all__ = ["GatedResidualRMSNorm", "GEGLU", "LayerNorm", "Linear", "MaskedSoftmax", "Mean", "PagedAttention", "RMSNorm",
           "ScaledDotProductAttention", "SlidingWindowAttention", "Softmax", "Sum", "Var", "VarMean"]


def _shape_tuple(shape: Union[int, Tuple[int, ...]]) -> Tuple[int, ...]:
    return (shape,) if isinstance(shape, int) else tuple(shape)


class _Projection(torch.nn.Module):
    """Shared parameter handling of Linear and GEGLU: weight [out, in], optional bias [out]."""

    def __init__(self, in_features, out_features, bias, use_accelerator, device, dtype):
        super().__init__()
        factory_kwargs = {"device": device, "dtype": dtype}
        self.in_features = in_features
        self.out_features = out_features
        self.use_accelerator = use_accelerator
        self.weight = torch.nn.Parameter(torch.empty(out_features, in_features, **factory_kwargs))
        if bias:
            self.bias = torch.nn.Parameter(torch.empty(out_features, **factory_kwargs))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def extra_repr(self):
        return (
            f"in_features={self.in_features}, "
            f"out_features={self.out_features}, "
            f"bias={self.bias is not None}, "
            f"backend=Trident"
        )


class GEGLU(_Projection):
    def __init__(
        self,
        in_features: int,
        out_features: int,
        bias: bool = True,
        use_accelerator: bool = False,
        device=None,
        dtype=None,
    ):
        """
        Linear projection to `out_features` columns followed by state * gelu(gate), where
        state is the first half of the projection and gate the second half; the output
        has out_features // 2 features (trident/module.py:299-364).
        """
        super().__init__(in_features, out_features, bias, use_accelerator, device, dtype)

    def forward(self, input: torch.Tensor):
        return function.geglu(input, self.weight, self.bias, self.use_accelerator)

    def reset_parameters(self):
        bound = math.sqrt(1 / self.in_features)
        util.uniform(self.weight, -bound, bound)
        if self.bias is not None:
            util.uniform(self.bias, -bound, bound)


class Linear(_Projection):
    def __init__(
        self,
        in_features: int,
        out_features: int,
        bias: bool = True,
        use_accelerator: bool = False,
        device=None,
        dtype=None,
    ):
        """y = x W^T + b (trident/module.py:764-826)."""
        super().__init__(in_features, out_features, bias, use_accelerator, device, dtype)

    def forward(self, input: torch.Tensor):
        return function.linear(input, self.weight, self.bias, self.use_accelerator)

    def reset_parameters(self):
        torch.nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))
        if self.bias is not None:
            fan_in, _ = util.calculate_fan_in_and_fan_out(self.weight)
            bound = 1 / math.sqrt(fan_in) if fan_in > 0 else 0
            util.uniform(self.bias, -bound, bound)


class LayerNorm(torch.nn.Module):
    def __init__(
        self,
        normalized_shape: Tuple[int, ...],
        eps: float = 1e-05,
        elementwise_affine: bool = True,
        device=None,
        dtype=None,
    ):
        """Layer normalisation over the trailing `normalized_shape` dimensions
        (trident/module.py:661-727); weight starts at one, bias at zero."""
        super().__init__()
        factory_kwargs = {"device": device, "dtype": dtype}
        self.normalized_shape = _shape_tuple(normalized_shape)
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        if elementwise_affine:
            self.weight = torch.nn.Parameter(torch.empty(self.normalized_shape, **factory_kwargs))
            self.bias = torch.nn.Parameter(torch.empty(self.normalized_shape, **factory_kwargs))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)
        self.reset_parameters()

    def forward(self, input: torch.Tensor):
        return function.layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)

    def reset_parameters(self):
        if self.elementwise_affine:
            util.fill(self.weight, 1)
            util.zero(self.bias)

    def extra_repr(self):
        return (
            f"{tuple(self.normalized_shape)},"
            f" eps={self.eps},"
            f" elementwise_affine={self.elementwise_affine},"
            f" backend=Trident"
        )


class RMSNorm(torch.nn.Module):
    def __init__(
        self,
        normalized_shape: Tuple[int, ...],
        p: float = -1.0,
        eps: float = 1e-05,
        bias: bool = False,
        device=None,
        dtype=None,
    ):
        """Root-mean-square normalisation of the last dimension; 0 <= p <= 1 takes the RMS
        over the leading int(p * width) features only (trident/module.py:998-1066)."""
        super().__init__()
        factory_kwargs = {"device": device, "dtype": dtype}
        self.normalized_shape = _shape_tuple(normalized_shape)
        self.p = p
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.empty(self.normalized_shape, **factory_kwargs))
        if bias:
            self.bias = torch.nn.Parameter(torch.empty(self.normalized_shape, **factory_kwargs))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def forward(self, input: torch.Tensor):
        return function.rms_norm(input, self.p, self.weight, self.bias, self.eps)

    def reset_parameters(self):
        util.fill(self.weight, 1.0)
        if self.bias is not None:
            util.zero(self.bias)

    def extra_repr(self):
        return (
            f"{tuple(self.normalized_shape)}, "
            f"p={self.p}, "
            f"eps={self.eps}, "
            f"bias={self.bias is not None}, "
            f"backend=Trident"
        )


class GatedResidualRMSNorm(torch.nn.Module):
    """Module form of function.gated_residual_rms_norm: the norm after a block (left out with
    post_norm=False), a gate with one value per feature (left out with gate=False; another gate can be
    passed to forward), the residual and the norm before the next block. Returns (output, residual)."""

    def __init__(
        self,
        normalized_shape: int,
        post_norm: bool = True,
        gate: bool = True,
        residual_scale: float = 1.0,
        eps: float = 1e-05,
        device=None,
        dtype=None,
    ):
        super().__init__()
        factory_kwargs = {"device": device, "dtype": dtype}
        self.normalized_shape = _shape_tuple(normalized_shape)
        self.residual_scale = residual_scale
        self.eps = eps
        for name, used in (("post_weight", post_norm), ("pre_weight", True), ("gate", gate)):
            if used:
                setattr(self, name, torch.nn.Parameter(torch.empty(self.normalized_shape, **factory_kwargs)))
            else:
                self.register_parameter(name, None)
        self.reset_parameters()

    def forward(self, input: torch.Tensor, residual: torch.Tensor, gate: torch.Tensor = None):
        return function.gated_residual_rms_norm(
            input,
            residual,
            self.post_weight,
            self.pre_weight,
            self.gate if gate is None else gate,
            self.residual_scale,
            self.eps,
        )

    def reset_parameters(self):
        for parameter in (self.post_weight, self.pre_weight, self.gate):
            if parameter is not None:
                util.fill(parameter, 1.0)

    def extra_repr(self):
        return (
            f"{tuple(self.normalized_shape)}, "
            f"post_norm={self.post_weight is not None}, "
            f"gate={self.gate is not None}, "
            f"residual_scale={self.residual_scale}, "
            f"eps={self.eps}, "
            f"backend=Trident"
        )


class ScaledDotProductAttention(torch.nn.Module):
    """Module form of function.scaled_dot_product_attention (the reference has only the function,
    trident/function/function.py:238-253). Dropout is active in training mode only."""

    def __init__(self, dropout_p: float = 0.0, is_causal: bool = False, use_accelerator: bool = False):
        super().__init__()
        self.dropout_p = dropout_p
        self.is_causal = is_causal
        self.use_accelerator = use_accelerator

    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, attn_mask: torch.Tensor = None):
        return function.scaled_dot_product_attention(
            query, key, value, attn_mask, self.dropout_p if self.training else 0.0, self.is_causal, self.use_accelerator
        )

    def extra_repr(self):
        return f"dropout_p={self.dropout_p}, is_causal={self.is_causal}, use_accelerator={self.use_accelerator}"


class SlidingWindowAttention(torch.nn.Module):
    """Module form of function.sliding_window_attention."""

    def __init__(self, window_size: int, num_sinks: int = 0, softmax_scale: float = None):
        super().__init__()
        self.window_size = window_size
        self.num_sinks = num_sinks
        self.softmax_scale = softmax_scale

    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor):
        return function.sliding_window_attention(
            query, key, value, self.window_size, self.num_sinks, self.softmax_scale
        )

    def extra_repr(self):
        return f"window_size={self.window_size}, num_sinks={self.num_sinks}, backend=Trident"


class PagedAttention(torch.nn.Module):
    """Keys and values of new tokens into the pages of a cache, then the tokens' attention over it
    (function.paged_cache_append and function.paged_attention with the same arguments)."""

    def __init__(self, window_size: int = None, num_sinks: int = 0, softmax_scale: float = None):
        super().__init__()
        self.window_size = window_size
        self.num_sinks = num_sinks
        self.softmax_scale = softmax_scale

    def forward(
        self,
        query: torch.Tensor,
        key: torch.Tensor,
        value: torch.Tensor,
        key_cache: torch.Tensor,
        value_cache: torch.Tensor,
        block_table: torch.Tensor,
        context_lengths: torch.Tensor,
        query_offsets: torch.Tensor = None,
        max_query_length: int = None,
        max_context_length: int = None,
    ):
        function.paged_cache_append(key, value, key_cache, value_cache, block_table, context_lengths, query_offsets)
        return function.paged_attention(
            query, key_cache, value_cache, block_table, context_lengths, query_offsets, max_query_length,
            max_context_length, self.window_size, self.num_sinks, self.softmax_scale,
        )

    def extra_repr(self):
        return f"window_size={self.window_size}, num_sinks={self.num_sinks}, backend=Trident"


class Softmax(torch.nn.Module):
    def __init__(self, dim: int = None):
        """Softmax of a 2-D input along `dim` (0 = down the columns, anything else = along
        the rows; trident/module.py:1141-1172)."""
        super().__init__()
        self.dim = dim

    def forward(self, input: torch.Tensor):
        return function.softmax(input, self.dim)

    def extra_repr(self):
        return f"dim={self.dim}, backend=Trident"


class MaskedSoftmax(torch.nn.Module):
    def __init__(self, dim: int = None):
        """Softmax that ignores the positions where `mask` is set (trident/module.py:829-861)."""
        super().__init__()
        self.dim = dim

    def forward(self, input: torch.Tensor, mask: torch.Tensor):
        return function.masked_softmax(input, mask, self.dim)

    def extra_repr(self):
        return f"dim={self.dim}, backend=Trident"


class Sum(torch.nn.Module):
    def __init__(self, dim: int = None):
        """Sum of a 2-D input along `dim` (0 = down the columns, anything else = along the rows;
        trident/module.py:1175-1197)."""
        super().__init__()
        self.dim = dim

    def forward(self, input: torch.Tensor):
        return function.sum(input, self.dim)

    def extra_repr(self):
        return f"dim={self.dim}, backend=Trident"


class Mean(torch.nn.Module):
    def __init__(self, dim: int = None):
        """Mean of a 2-D input along `dim` (trident/module.py:898-920)."""
        super().__init__()
        self.dim = dim

    def forward(self, input: torch.Tensor):
        return function.mean(input, self.dim)

    def extra_repr(self):
        return f"dim={self.dim}, backend=Trident"


class Var(torch.nn.Module):
    def __init__(self, dim: int = None, correction: int = 1):
        """Variance of a 2-D input along `dim`, divided by n - correction (trident/module.py:1209-1233)."""
        super().__init__()
        self.dim = dim
        self.correction = correction

    def forward(self, input: torch.Tensor):
        return function.var(input, self.dim, self.correction)

    def extra_repr(self):
        return f"dim={self.dim}, correction={self.correction}, backend=Trident"


class VarMean(torch.nn.Module):
    def __init__(self, dim: int = None, correction: int = 1):
        """Variance and mean of a 2-D input along `dim` (trident/module.py:1245-1269)."""
        super().__init__()
        self.dim = dim
        self.correction = correction

    def forward(self, input: torch.Tensor):
        return function.var_mean(input, self.dim, self.correction)

    def extra_repr(self):
        return f"dim={self.dim}, correction={self.correction}, backend=Trident"
