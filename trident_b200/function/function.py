"""Functional API with the signatures of trident/function/function.py for the operations
this library implements."""

import math

import torch

from trident_b200 import operation, util

__all__ = [
    "gated_residual_rms_norm",
    "geglu",
    "layer_norm",
    "linear",
    "masked_softmax",
    "rms_norm",
    "rms_norm_geglu",
    "mean",
    "paged_attention",
    "paged_cache_append",
    "scaled_dot_product_attention",
    "sliding_window_attention",
    "softmax",
    "sum",
    "var",
    "var_mean",
]


def gated_residual_rms_norm(
    input: torch.Tensor,
    residual: torch.Tensor,
    post_weight: torch.Tensor = None,
    pre_weight: torch.Tensor = None,
    gate: torch.Tensor = None,
    residual_scale: float = 1.0,
    eps: float = 1e-08,
):
    """
    Applies the step between two blocks of a transformer (not in the reference): the norm after a block,
    its gate, the scaled residual and the norm before the next block.

        output_residual = residual_scale * residual + gate * rms_norm(input, -1.0, post_weight)
        output = rms_norm(output_residual, -1.0, pre_weight)

    Without post_weight the input is not normalised, without gate it is not scaled. The gate holds one
    value per feature ([features]), or has the dimensions of the input with ones from some dimension on
    ([batch, 1, features]: one vector per sequence). Returns (output, output_residual).

    See GatedResidualRMSNorm for details.
    """
    args = (input, residual, post_weight, pre_weight, gate, residual_scale, eps)
    if util.needs_grad(input, residual, post_weight, pre_weight, gate):
        return operation.GatedResidualRMSNorm.apply(*args)
    return operation.GatedResidualRMSNorm.run(*args, statistics=False)[0]


def geglu(input: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor = None, use_accelerator: bool = False):
    """
    Applies GEGLU to an input.

    See GEGLU for details.
    """
    if input.dim() == 2:
        output = operation.GEGLU.apply(input.view(1, *input.shape), weight, bias, use_accelerator)
        return output.view(output.shape[1:3])
    else:
        return operation.GEGLU.apply(input, weight, bias, use_accelerator)


def layer_norm(input, normalized_shape, weight=None, bias=None, eps=1e-05):
    """
    Applies Layer Normalization for last certain number of dimensions.

    See LayerNorm for details.
    """
    if isinstance(normalized_shape, int):
        normalized_shape = (normalized_shape,)
    return operation.LayerNorm.apply(input, tuple(normalized_shape), weight, bias, eps)


def linear(
    input: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor = None,
    use_accelerator: bool = False,
):
    """
    Applies Linear Transformation to an input.

    See Linear for more details.
    """
    if input.dim() == 2:
        output = operation.Linear.apply(input.view(1, *input.shape), weight, bias, use_accelerator)
        return output.view(output.shape[1:3])
    else:
        return operation.Linear.apply(input, weight, bias, use_accelerator)


def masked_softmax(input: torch.Tensor, mask: torch.Tensor, dim: int):
    """
    Applies Masked Softmax to an input rescaling them so that an output lie in the range [0,1] and sum to 1.

    See MaskedSoftmax for more details.
    """
    return operation.MaskedSoftmax.apply(input, mask, dim)


def rms_norm(input: torch.Tensor, p: float, weight: torch.Tensor, bias: torch.Tensor = None, eps: float = 1e-08):
    """
    Applies Root Mean Square Layer Normalization to an input.

    See RMSNorm for details.
    """
    return operation.RMSNorm.apply(input.view(-1, input.shape[-1]), p, weight, bias, eps).view(input.shape)


def rms_norm_geglu(
    input: torch.Tensor,
    p: float,
    norm_weight: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor = None,
    eps: float = 1e-08,
    folded_weight: torch.Tensor = None,
):
    """
    geglu(rms_norm(input, p, norm_weight, None, eps), weight, bias) as one operation (not in the
    reference): the normalised input is never written to memory in the forward pass.

    `folded_weight`, if given, must equal weight * norm_weight (computed once by the caller while
    both stay fixed); otherwise it is formed on every call.
    """
    shape = input.shape
    out = operation.RMSNormGEGLU.apply(input.reshape(-1, shape[-1]), p, norm_weight, weight, bias, eps, folded_weight)
    return out.view(*shape[:-1], out.shape[-1])


def paged_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lengths: torch.Tensor,
    query_offsets: torch.Tensor = None,
    max_query_length: int = None,
    max_context_length: int = None,
    window_size: int = None,
    num_sinks: int = 0,
    softmax_scale: float = None,
    output: torch.Tensor = None,
):
    """
    Computes attention of each sequence's newest tokens over the keys and values of a paged cache (not in
    the reference): one token per sequence, or a chunk of a prompt, in one call.

    key_cache and value_cache are [pages, page size, key heads, head size]; the key at position x of
    sequence s is row x % page size of page block_table[s][x // page size]. context_lengths counts the
    keys of each sequence, its new tokens included (paged_cache_append writes them first, with the same
    arguments). The new tokens of sequence s are rows query_offsets[s] to query_offsets[s + 1] of query
    [tokens, heads, head size]; without query_offsets there is one per sequence. A token sees the positions
    up to its own; with window_size, those less than window_size back and the first num_sinks, and table
    entries of blocks that no token sees may be anything. block_table, context_lengths and query_offsets
    are int32 tensors on the device and are not read by the host. A context longer than the table has room for keeps
    its positions: the keys behind the table do not exist, and are not written by paged_cache_append.

    Of each sequence the first max_query_length new tokens are computed (default: all of them);
    max_context_length is the longest context expected (default: what the table holds) and only chooses how
    the work is split. Both have to be given for the best speed, and stay what they are in a captured graph.
    Rows of query that belong to no sequence or lie beyond max_query_length give zeros, or leave `output`, where it
    is given, as it was.
    What pages hold beyond a context is not read into any result; keys and values inside it have to be finite.
    """
    scale = 1.0 / math.sqrt(query.shape[-1]) if softmax_scale is None else softmax_scale
    return operation.paged_attention(
        query, key_cache, value_cache, block_table, context_lengths, query_offsets, max_query_length,
        max_context_length, window_size, num_sinks, scale, output,
    )


def paged_cache_append(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lengths: torch.Tensor,
    query_offsets: torch.Tensor = None,
):
    """
    Writes the keys and values [tokens, key heads, head size] of new tokens into the pages of a cache, in
    place: the i-th of t new tokens of a sequence goes to position context_length - t + i. Sequences may share
    pages, but not one that both write: of two tokens written to one place either may stay.

    See paged_attention for the other arguments.
    """
    operation.paged_cache_append(key, value, key_cache, value_cache, block_table, context_lengths, query_offsets)


def scaled_dot_product_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    attn_mask: torch.Tensor = None,
    dropout_p: float = 0.0,
    is_causal: bool = False,
    use_accelerator: bool = False,
):
    """
    Computes scaled dot product attention on query, key and value tensors,
    and applying dropout if a probability greater than 0.0 is specified.

    The softmax scale is 1/sqrt(head size). attn_mask is additive (any float type) or boolean
    (True = attend). Dropout acts on the attention output, where the reference applies it.
    """
    return operation.Attention.apply(
        query, key, value, attn_mask, dropout_p, is_causal, 1.0 / math.sqrt(key.shape[-1]), use_accelerator
    )


def sliding_window_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    window_size: int,
    num_sinks: int = 0,
    softmax_scale: float = None,
):
    """
    Computes causal attention in which a query sees its last window_size positions (its own among them)
    and the first num_sinks tokens (not in the reference, whose attention is dense).

    query is [batch, heads, length, head size], key and value [batch, key heads, length, head size]; each
    key head serves heads / key heads consecutive query heads. The softmax scale is 1/sqrt(head size)
    unless given. Any strides are taken; the output is laid out as query is. Keys and values have to be
    finite, those of padding too: what a query does not see has the weight 0, and 0 times NaN is NaN.

    See WindowAttention for more details.
    """
    scale = 1.0 / math.sqrt(query.shape[-1]) if softmax_scale is None else softmax_scale
    if util.needs_grad(query, key, value):
        return operation.WindowAttention.apply(query, key, value, window_size, num_sinks, scale)
    return operation.WindowAttention.run(query, key, value, window_size, num_sinks, scale, statistics=False)[0]


def softmax(input: torch.Tensor, dim: int = None):
    """
    Applies Softmax to an input rescaling them so that an output lie in the range [0,1] and sum to 1.

    See Softmax for more details.
    """
    return operation.Softmax.apply(input, dim)


def sum(input: torch.Tensor, dim=None):
    """
    Returns the sum along the specified dimension in an input.

    See Sum for more details.
    """
    return operation.Sum.apply(input, dim)


def mean(input: torch.Tensor, dim=None):
    """
    Returns the mean along the specified dimension in an input.

    See Mean for more details.
    """
    return operation.Mean.apply(input, dim)


def var(input: torch.Tensor, dim=None, correction: int = 1):
    """
    Returns the variance along the specified dimension in an input.

    See Var for more details.
    """
    return operation.Var.apply(input, dim, correction)


def var_mean(input: torch.Tensor, dim=None, correction: int = 1):
    """
    Returns the variance and mean along the specified dimension in an input.

    See VarMean for more details.
    """
    return operation.VarMean.apply(input, dim, correction)
