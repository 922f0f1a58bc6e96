"""Differentiable dense operators on the matrix cores of the GPU.

  linear_act      y = act(x W^T + b) + r in one launch, and its gradients
  grouped_linear  the same with one W and b for each group of rows: a cohort of
                  client models side by side, each on its own number of samples

Both take float32, bfloat16 or float16 HIP tensors (one type a call; sums are
float32, or better, and rounded once) of any strides and raise for anything
else.  float32 products have float32's accuracy.  The value before the activation
is kept for the gradient in the tensors' type.

A backward pass may be captured into a graph together with its forward pass;
as with any torch operator, no eager graph of the same leaves may be alive then.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import train_ops

__all__ = ["grouped_linear", "linear_act"]


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, offsets, activation):
        # relu's gradient can be told from its output; the others need z
        inner = any(ctx.needs_input_grad[:3])
        want_z = inner and activation != "none" and (activation != "relu" or residual is not None)
        y, z = train_ops.product_forward(x, weight, bias, residual, activation, offsets, want_z)
        keep = None if not inner or activation == "none" else z if want_z else y
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None,
                              weight if ctx.needs_input_grad[0] else None, offsets, keep)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, offsets, keep = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            dz = dy if keep is None else train_ops.act_backward(dy, keep, ctx.activation)
            if need_x:
                dx = train_ops.product_grad_input(dz, weight, offsets)
            if need_w or need_b:
                dw, db = train_ops.product_grad_weight(dz, x if need_w else dz, offsets, need_w,
                                                       need_b)
        return dx, dw, db, dy if need_r else None, None, None


def _apply(x, weight, bias, residual, offsets, activation):
    if torch.is_grad_enabled() and any(
            isinstance(t, torch.Tensor) and t.requires_grad for t in (x, weight, bias, residual)):
        return _Product.apply(x, weight, bias, residual, offsets, activation)
    return train_ops.product_forward(x, weight, bias, residual, activation, offsets)[0]


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None,
               activation: str = "none") -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: ``x`` [..., in], ``weight`` [out, in],
    ``bias`` [out], ``residual`` [..., out]; ``activation`` is ``"none"``,
    ``"relu"``, ``"gelu"`` (erf) or ``"silu"``."""
    train_ops._require(x, "x")
    train_ops._require(weight, "weight", x)
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit "
                         "[..., in] and [out, in]")
    lead = x.shape[:-1]
    if residual is not None:
        train_ops._require(residual, "residual", x)
        if residual.shape != (*lead, weight.shape[0]):
            raise ValueError(f"residual must have shape {(*lead, weight.shape[0])}, "
                             f"got {tuple(residual.shape)}")
    n = lead.numel()
    y = _apply(x.reshape(n, x.shape[-1]), weight, bias,
               None if residual is None else residual.reshape(n, weight.shape[0]), None,
               activation)
    return y if len(lead) == 1 else y.view(*lead, weight.shape[0])


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                   bias: Optional[torch.Tensor] = None,
                   residual: Optional[torch.Tensor] = None,
                   activation: str = "none") -> torch.Tensor:
    """Rows ``offsets[g] .. offsets[g + 1]`` of the result are
    ``act(x @ weight[g].T + bias[g]) + residual``: ``x`` [N, in], ``weight``
    [G, out, in], ``bias`` [G, out], ``residual`` [N, out], ``offsets`` [G + 1]
    ascending int32 or int64 on the device (they are not read on the host; one
    outside 0 .. N is cut to it).  A group may be empty; a row in no group gets
    its residual, or zero, and its x no gradient.

    ``weight`` may be a view with any group and row stride, such as a layer of K
    models whose flat vectors are the rows of one slab."""
    if offsets is None:
        raise TypeError("offsets must be a torch.Tensor")
    return _apply(x, weight, bias, residual, offsets, activation)
