"""Host-side helpers of the operation layer; counterparts of trident/util/util.py."""

import torch
from torch.autograd import forward_ad

from trident_b200 import config

__all__ = [
    "calculate_fan_in_and_fan_out",
    "fill",
    "first_order",
    "is_pow2",
    "is_watched",
    "needs_grad",
    "size_and_stride",
    "push_trace",
    "pop_trace",
    "written",
    "uniform",
    "zero",
]


def calculate_fan_in_and_fan_out(input: torch.Tensor):
    with torch.no_grad():
        return torch.nn.init._calculate_fan_in_and_fan_out(input)


def fill(inp, val):
    with torch.no_grad():
        return inp.fill_(val)


def is_pow2(value):
    """True for 1, 2, 4, ... (trident/util/util.py:61-62)."""
    return value != 0 and (value & (value - 1)) == 0


# (looked up once: the calls that ask take 10 us of host time in all)
_increment_version = torch.autograd.graph.increment_version
_tracing_state = torch._C._get_tracing_state
_transforms_active = torch._C._are_functorch_transforms_active


def needs_grad(*tensors):
    """Whether an operation on these tensors (None allowed) has to go through its autograd Function: autograd
    would record it, or something else that only sees Functions is looking on."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return is_watched()


class _FirstOrder(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, count, *tensors):
        ctx.what = what
        return tuple(t.view_as(t) for t in tensors[:count])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.what} has no second derivative.")


def first_order(what, grads, *sources):
    """The gradients (None allowed) of a backward pass that cannot be differentiated itself, computed from `sources`.
    Under create_graph=True they are tied to these by a node that refuses: without one a second derivative would
    lose their part of a sum without a word."""
    if not torch.is_grad_enabled():
        return grads
    given = [g for g in grads if g is not None]
    tied = iter(_FirstOrder.apply(what, len(given), *given, *(t for t in sources if t is not None)))
    return tuple(None if g is None else next(tied) for g in grads)


def written(*tensors):
    """Tells autograd that these tensors were written in place by a kernel: a graph that saved one of them refuses its
    backward pass, as after an in-place operation of torch. (Inference tensors are never saved and keep no version.)"""
    try:
        _increment_version(tensors)
    except RuntimeError:  # (an inference tensor outside of inference mode)
        _increment_version([t for t in tensors if not t.is_inference()])


def is_watched():
    """Whether a trace, a function transform or forward-mode differentiation is under way: they would take the
    output of a kernel that is called directly for an empty tensor, or for one without a tangent."""
    return _tracing_state() is not None or _transforms_active() or forward_ad._current_level >= 0


def size_and_stride(input: torch.Tensor, dim: int):
    """(rows, cols, row_stride, col_stride) of a 2-D tensor reduced along `dim`.

    dim == 0 reduces down the columns, every other value along the last dimension
    (trident/util/util.py:65-77). Only 2-D inputs are accepted: the reference's 3-D
    branch returns six values that none of its row operations can unpack.
    """
    if input.dim() != 2:
        raise ValueError(f"{dim} is not supported.")
    if dim == 0:
        x_size, y_size = input.shape
        return y_size, x_size, input.stride(1), input.stride(0)
    y_size, x_size = input.shape
    return y_size, x_size, input.stride(0), input.stride(1)


def push_trace(message: str):
    """Opens an NVTX range when config.use_trace is set (trident/util/util.py:93-95)."""
    if config.use_trace and torch.cuda.is_available():
        torch.cuda.nvtx.range_push(message)


def pop_trace():
    if config.use_trace and torch.cuda.is_available():
        torch.cuda.nvtx.range_pop()


def uniform(input: torch.Tensor, a: float = 0.0, b: float = 1.0):
    with torch.no_grad():
        return torch.nn.init.uniform_(input, a, b)


def zero(inp):
    with torch.no_grad():
        return inp.zero_()
