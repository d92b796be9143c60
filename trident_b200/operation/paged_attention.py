"""Attention over a paged cache and the write into it, over libtb200 (not in the reference, which has no
serving path). Neither has a backward pass."""

import torch

from trident_b200 import _lib, util
from trident_b200.operation.window_attention import check_heads, check_window

MOST_TOKENS = 2 ** 30 - 1


def _check_cache(key_cache, value_cache, block_table, context_lengths, query_offsets, tokens, tensors):
    if key_cache.dim() != 4 or value_cache.dim() != 4:
        raise ValueError("The dimension of key_cache and value_cache should be 4: [pages, page size, heads, head size].")
    if key_cache.shape != value_cache.shape:
        raise ValueError("key_cache and value_cache should have the same shape.")
    if key_cache.shape[1] == 0:
        raise ValueError("A page should hold at least one token.")
    if block_table.dim() != 2 or context_lengths.dim() != 1 or block_table.shape[0] != context_lengths.shape[0]:
        raise ValueError("block_table should be [sequences, blocks] and context_lengths [sequences].")
    if query_offsets is None:
        if tokens != block_table.shape[0]:
            raise ValueError("Without query_offsets there should be one new token per sequence.")
    elif query_offsets.dim() != 1 or query_offsets.shape[0] != block_table.shape[0] + 1:
        raise ValueError("query_offsets should be [sequences + 1].")
    for tensor in (block_table, context_lengths, query_offsets):
        if tensor is not None and tensor.dtype != torch.int32:
            raise ValueError(
                "block_table, context_lengths and query_offsets should have the dtype torch.int32."
            )
    grad = key_cache.requires_grad or value_cache.requires_grad
    dtype = key_cache.dtype
    same = value_cache.dtype == dtype
    for tensor in tensors.values():
        same = same and tensor.dtype == dtype
        grad = grad or tensor.requires_grad
    if not same:
        raise ValueError(f"{', '.join(tensors)}, key_cache and value_cache should have the same dtype.")
    _lib.dtype_code(dtype)
    if grad and torch.is_grad_enabled():
        raise ValueError("Paged attention has no backward pass: call it under torch.no_grad().")
    if util.is_watched():
        _check_unwatched(key_cache, value_cache, *tensors.values())


def _check_unwatched(*tensors):
    if torch._C._get_tracing_state() is not None:
        raise ValueError("Paged attention cannot be traced: a trace records no call of the library.")
    if torch._C._are_functorch_transforms_active():
        raise ValueError("Paged attention cannot be called under function transforms (vmap, jvp, ...).")
    if any(torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("Paged attention has no forward-mode derivative.")


def _check_room(block_table, key_cache):
    if block_table.shape[1] == 0 or key_cache.shape[0] == 0:
        raise ValueError("block_table should have a block for every sequence and the cache at least one page.")


def _check_written(name, tensor):
    """A tensor that is written must have a place of its own for each element."""
    if 0 in tensor.stride() and any(st == 0 and size > 1 for st, size in zip(tensor.stride(), tensor.shape)):
        raise ValueError(f"{name} should not be expanded: some of its elements share their memory.")


def _index(tensor):
    """An int32 tensor whose last dimension is dense."""
    return tensor if tensor is None or tensor.numel() == 0 or tensor.stride(-1) == 1 else tensor.contiguous()


def paged_attention(
    query,
    key_cache,
    value_cache,
    block_table,
    context_lengths,
    query_offsets,
    max_query_length,
    max_context_length,
    window_size,
    num_sinks,
    softmax_scale,
    output,
):
    if query.dim() != 3:
        raise ValueError("The dimension of query should be 3: [tokens, heads, head size].")
    tokens, heads, x_size = query.shape
    tensors = {"query": query} if output is None else {"query": query, "output": output}
    _check_cache(key_cache, value_cache, block_table, context_lengths, query_offsets, tokens, tensors)
    if key_cache.shape[-1] != x_size:
        raise ValueError("query and key_cache should have the same head size.")
    check_heads(heads, key_cache.shape[2], x_size)
    if window_size is None:
        if num_sinks != 0:
            raise ValueError("num_sinks needs a window_size.")
    else:
        check_window(window_size, num_sinks)
    if output is not None and output.shape != query.shape:
        raise ValueError("output and query should have the same shape.")
    if output is not None:
        _check_written("output", output)
    if query_offsets is None:
        max_query_length = 1
    elif max_query_length is None:
        max_query_length = tokens
    elif max_query_length < 0:
        raise ValueError("max_query_length should not be negative.")
    room = block_table.shape[1] * key_cache.shape[1]
    if max_context_length is None or max_context_length > room:
        max_context_length = room
    elif max_context_length < 0:
        raise ValueError("max_context_length should not be negative.")
    _lib.require_one_device(
        key_cache, value_cache, block_table, context_lengths, query_offsets, *tensors.values()
    )
    max_query_length = max(1, min(max_query_length, tokens, MOST_TOKENS))
    max_context_length = min(max_context_length, MOST_TOKENS)
    sequences = block_table.shape[0]
    zero_rest = output is None and query_offsets is not None
    if sequences == 0 or tokens == 0:
        return torch.zeros_like(query) if output is None else output
    _check_room(block_table, key_cache)
    given = output is not None
    if not given:
        output = torch.empty_like(query)
    window = 0 if window_size is None else min(window_size, MOST_TOKENS)
    sinks = min(num_sinks, MOST_TOKENS)

    util.push_trace("PagedAttention")
    size = _lib.paged_attention_workspace(
        query, key_cache.shape[2], sequences, max_query_length, max_context_length, window, sinks
    )
    workspace = torch.empty(size, dtype=torch.uint8, device=query.device) if size else None
    util.push_trace("tb200_paged_attention")
    _lib.paged_attention(
        output,
        query,
        key_cache,
        value_cache,
        _index(block_table),
        _index(context_lengths),
        _index(query_offsets),
        workspace,
        max_query_length,
        max_context_length,
        window,
        sinks,
        softmax_scale,
        zero_rest,
    )
    if given:
        util.written(output)
    util.pop_trace()
    util.pop_trace()

    return output


def paged_cache_append(key, value, key_cache, value_cache, block_table, context_lengths, query_offsets):
    if key.dim() != 3 or key.shape != value.shape:
        raise ValueError("key and value should have the same shape [tokens, heads, head size].")
    tensors = {"key": key, "value": value}
    _check_cache(key_cache, value_cache, block_table, context_lengths, query_offsets, key.shape[0], tensors)
    if key.shape[1:] != key_cache.shape[2:]:
        raise ValueError("key and key_cache should have the same heads and head size.")
    check_heads(key.shape[1], key.shape[1], key.shape[2])
    _check_written("key_cache", key_cache)
    _check_written("value_cache", value_cache)
    _lib.require_one_device(
        key_cache, value_cache, block_table, context_lengths, query_offsets, *tensors.values()
    )
    if key.shape[0] == 0 or block_table.shape[0] == 0:
        return
    _check_room(block_table, key_cache)

    util.push_trace("tb200_paged_cache_append")
    _lib.paged_cache_append(
        key_cache, value_cache, key, value, _index(block_table), _index(context_lengths), _index(query_offsets)
    )
    util.written(key_cache, value_cache)
    util.pop_trace()
