"""Gated residual RMSNorm autograd Function over libtb200 (not in the reference, which has RMSNorm alone,
trident/operation/rms_norm.py)."""

from typing import Any

import torch

from trident_b200 import _lib, util


def rows_per_gate(input: torch.Tensor, gate: torch.Tensor) -> int:
    """How many rows of `input` share one gate vector: 0 for one vector in all. `gate` has the features
    of `input` and, if more dimensions, the leading dimensions of `input` with ones from some
    dimension on."""
    if gate.dim() == 1 and gate.shape[0] == input.shape[-1]:
        return 0
    if gate.shape[-1:] != input.shape[-1:]:
        raise ValueError(f"A gate of shape {tuple(gate.shape)} does not fit an input of shape {tuple(input.shape)}.")
    if gate.dim() != input.dim():
        raise ValueError(f"A gate of shape {tuple(gate.shape)} does not fit an input of shape {tuple(input.shape)}.")
    lead, wanted = gate.shape[:-1], input.shape[:-1]
    own = 0
    while own < len(lead) and lead[own] == wanted[own]:
        own += 1
    if any(size != 1 for size in lead[own:]):
        raise ValueError(f"A gate of shape {tuple(gate.shape)} does not fit an input of shape {tuple(input.shape)}.")
    vectors = 1
    for size in lead:
        vectors *= size
    if vectors <= 1:
        return 0
    rows = 1
    for size in wanted:
        rows *= size
    return rows // vectors


class GatedResidualRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, *args: Any, **kwargs: Any):
        outputs, saved, group = GatedResidualRMSNorm.run(*args)

        ctx.save_for_backward(*saved)
        ctx.set_materialize_grads(False)
        ctx.group = group
        ctx.residual_scale = args[5]
        ctx.eps = args[6]

        return outputs

    @staticmethod
    def run(input, residual, post_weight, pre_weight, gate, residual_scale, eps, statistics=True):
        """The forward pass: ((output, output_residual), what the backward pass needs, rows per gate). Without
        `statistics` the rms of the rows is not kept."""
        shape = input.shape
        if len(shape) < 1 or shape[-1] == 0:
            raise ValueError("input should have at least one feature.")
        if residual.shape != shape:
            raise ValueError("input and residual should have the same shape.")
        if pre_weight is None:
            raise ValueError("pre_weight should be given.")
        x_size = shape[-1]
        for weight in (post_weight, pre_weight):
            if weight is not None and (weight.dim() != 1 or weight.shape[0] != x_size):
                raise ValueError(f"A weight should have the shape ({x_size},), got {tuple(weight.shape)}.")
        group = 0 if gate is None else rows_per_gate(input, gate)
        for tensor in (residual, post_weight, pre_weight, gate):
            if tensor is not None and tensor.dtype != input.dtype:
                raise ValueError("input, residual, weights and gate should have the same dtype.")
        _lib.dtype_code(input.dtype)
        _lib.require_one_device(input, residual, post_weight, pre_weight, gate)

        util.push_trace("GatedResidualRMSNorm.__forward")
        input, residual, pre_weight = input.contiguous(), residual.contiguous(), pre_weight.contiguous()
        post_weight = None if post_weight is None else post_weight.contiguous()
        gate = None if gate is None else gate.contiguous()
        y_size = input.numel() // x_size
        output, output_residual = torch.empty_like(input), torch.empty_like(input)
        rms = torch.empty(2, y_size, device=input.device, dtype=torch.float32) if statistics else None

        util.push_trace("tb200_gated_residual_rms_norm_fwd")
        _lib.gated_residual_rms_norm_fwd(
            output,
            output_residual,
            rms,
            input,
            residual,
            post_weight,
            pre_weight,
            gate,
            y_size,
            x_size,
            group,
            residual_scale,
            eps,
        )
        util.pop_trace()
        util.pop_trace()

        return (output, output_residual), (input, residual, post_weight, pre_weight, gate, rms), group

    @staticmethod
    def backward(ctx: Any, *grad_outputs: Any):
        grad_output, grad_output_residual = grad_outputs
        if grad_output is None and grad_output_residual is None:
            return (None,) * 7

        util.push_trace("GatedResidualRMSNorm.__backward")
        grads = GatedResidualRMSNorm.__backward(
            grad_output,
            grad_output_residual,
            *ctx.saved_tensors,
            ctx.needs_input_grad,
            ctx.group,
            ctx.residual_scale,
            ctx.eps,
        )
        util.pop_trace()

        grads = util.first_order("Gated residual RMSNorm", grads, *grad_outputs, *ctx.saved_tensors)

        return (*grads, None, None)

    @staticmethod
    def __backward(grad_output, grad_output_residual, input, residual, post_weight, pre_weight, gate, rms, needs,
                   group, residual_scale, eps):
        """One pass over the rows, and one launch that adds the parts of the weight and gate gradients."""
        x_size = input.shape[-1]
        y_size = input.numel() // x_size
        grad_output, grad_output_residual = (
            None if t is None else t.contiguous() for t in (grad_output, grad_output_residual)
        )
        grad_input, grad_residual = torch.empty_like(input), torch.empty_like(input)
        if y_size == 0:  # sums over no rows
            return grad_input, grad_residual, *(
                torch.zeros_like(t) if t is not None and need else None
                for t, need in zip((post_weight, pre_weight, gate), needs[2:5])
            )
        grad_post_weight, grad_pre_weight, grad_gate = (
            torch.empty_like(t) if t is not None and need else None
            for t, need in zip((post_weight, pre_weight, gate), needs[2:5])
        )
        workspace = None
        if any(t is not None for t in (grad_post_weight, grad_pre_weight, grad_gate)):
            workspace = torch.empty(
                max(_lib.gated_residual_rms_norm_bwd_workspace(input, y_size, x_size, group), 16),
                dtype=torch.uint8,
                device=input.device,
            )

        util.push_trace("tb200_gated_residual_rms_norm_bwd")
        _lib.gated_residual_rms_norm_bwd(
            grad_input,
            grad_residual,
            grad_post_weight,
            grad_pre_weight,
            grad_gate,
            grad_output,
            grad_output_residual,
            input,
            residual,
            post_weight,
            pre_weight,
            gate,
            rms,
            workspace,
            y_size,
            x_size,
            group,
            residual_scale,
            eps,
        )
        util.pop_trace()

        return grad_input, grad_residual, grad_post_weight, grad_pre_weight, grad_gate
