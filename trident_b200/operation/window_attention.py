"""Window attention autograd Function over libtb200 (not in the reference, whose attention is dense,
trident/operation/attention.py)."""

from typing import Any

import torch

from trident_b200 import _lib, util

HEAD_SIZES = (16, 32, 64, 128)


def check_window(window_size, num_sinks):
    if isinstance(window_size, bool) or not isinstance(window_size, int) or window_size < 1:
        raise ValueError(f"window_size should be a positive integer, got {window_size}.")
    if isinstance(num_sinks, bool) or not isinstance(num_sinks, int) or num_sinks < 0:
        raise ValueError(f"num_sinks should be a non-negative integer, got {num_sinks}.")


def check_heads(heads, kv_heads, size):
    if kv_heads == 0 or heads % kv_heads != 0:
        raise ValueError(f"The number of query heads ({heads}) should be a multiple of that of key heads ({kv_heads}).")
    if heads == 0 or heads // kv_heads > 64:
        raise ValueError("A key head should have 1 to 64 query heads.")
    if size not in HEAD_SIZES:
        raise ValueError(f"The head size should be one of {HEAD_SIZES}, got {size}.")


class WindowAttention(torch.autograd.Function):
    """Causal attention in which a query at position i sees the keys j <= i with i - j < window_size or
    j < num_sinks. No atomics: the same inputs give the same output and gradients, bit for bit."""

    @staticmethod
    def forward(ctx: Any, *args: Any, **kwargs: Any):
        output, low, log_sum_exp, window_size, num_sinks = WindowAttention.run(*args)

        ctx.save_for_backward(*args[:3], output, low, log_sum_exp)
        ctx.window_size = window_size
        ctx.num_sinks = num_sinks
        ctx.softmax_scale = args[5]

        return output

    @staticmethod
    def run(query, key, value, window_size, num_sinks, softmax_scale, statistics=True):
        """The forward pass: (output, what its rounding to 16 bits left, log-sum-exp of every score row, window and
        sinks cut to the length). Without `statistics`, and the second of 32-bit operands, those of backward are None."""
        if query.dim() != 4 or key.dim() != 4 or value.dim() != 4:
            raise ValueError("The dimension of query, key and value should be 4.")
        if key.shape != value.shape:
            raise ValueError("key and value should have the same shape.")
        batch, heads, y_size, x_size = query.shape
        key_batch, kv_heads, key_length, key_size = key.shape
        if key_batch != batch or key_length != y_size or key_size != x_size:
            raise ValueError("query and key should have the same batch, length and head size.")
        check_heads(heads, kv_heads, x_size)
        check_window(window_size, num_sinks)
        if query.dtype != key.dtype or query.dtype != value.dtype:
            raise ValueError("query, key and value should have the same dtype.")
        _lib.dtype_code(query.dtype)
        _lib.require_one_device(query, key, value)
        # beyond the length of the sequence both mean the same (and any integer fits the library's types)
        window_size, num_sinks = min(window_size, max(y_size, 1)), min(num_sinks, y_size)

        util.push_trace("WindowAttention.__forward")
        output = torch.empty_like(query)  # laid out as query is
        low = log_sum_exp = None
        if statistics:
            if query.dtype != torch.float32:
                low = torch.empty_like(output)
            log_sum_exp = torch.empty((batch, heads, y_size), device=query.device, dtype=torch.float32)
        util.push_trace("tb200_window_attention_fwd")
        _lib.window_attention_fwd(output, log_sum_exp, query, key, value, window_size, num_sinks, softmax_scale, low)
        util.pop_trace()
        util.pop_trace()

        return output, low, log_sum_exp, window_size, num_sinks

    @staticmethod
    def backward(ctx: Any, *grad_outputs: Any):
        (grad_output,) = grad_outputs

        util.push_trace("WindowAttention.__backward")
        grads = WindowAttention.__backward(
            grad_output, *ctx.saved_tensors, ctx.window_size, ctx.num_sinks, ctx.softmax_scale
        )
        util.pop_trace()

        return (*util.first_order("Window attention", grads, grad_output, *ctx.saved_tensors), None, None, None)

    @staticmethod
    def __backward(grad_output, query, key, value, output, low, log_sum_exp, window_size, num_sinks, softmax_scale):
        """delta, dq, dk and dv (and, with sinks, the sum of their parts)."""
        if 0 in grad_output.stride():
            # (an expanded gradient, as that of a sum: the kernels read whole rows)
            grad_output = grad_output.contiguous()
        grad_query, grad_key, grad_value = (torch.empty_like(t) for t in (query, key, value))
        workspace = torch.empty(
            max(_lib.window_attention_bwd_workspace(query, key, window_size, num_sinks), 16),
            dtype=torch.uint8,
            device=query.device,
        )

        util.push_trace("tb200_window_attention_bwd")
        _lib.window_attention_bwd(
            grad_query,
            grad_key,
            grad_value,
            grad_output,
            query,
            key,
            value,
            output,
            log_sum_exp,
            workspace,
            window_size,
            num_sinks,
            softmax_scale,
            low,
        )
        util.pop_trace()

        return grad_query, grad_key, grad_value
