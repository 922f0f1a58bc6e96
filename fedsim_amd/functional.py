"""Differentiable dense operators on the matrix cores of the GPU.

  linear_act      y = act(x W^T + b) + r in one launch, and its gradients
  grouped_linear  the same with one W and b for each group of rows: a cohort of
                  client models side by side, each on its own number of samples

Both take float32, bfloat16 or float16 HIP tensors (one type a call; sums are
float32, or better, and rounded once) of any strides and raise for anything
else.  A float32 product of two values is good to 2^-24 of itself, as float32's
own, before it is added up; a factor below 2^-110 may lose its part below 2^-125.
The value before the activation is kept for the gradient in the tensors' type, and
so is the gradient there, dz, for the products that make dx and dW: in 16 bits these
are off by about 1.5 of their own roundings.  db is summed from dz unrounded.

A backward pass may be captured into a graph together with its forward pass;
as with any torch operator, no eager graph of the same leaves may be alive then.
They can be differentiated once, and cannot be traced (torch.jit.trace, make_fx,
torch.export); torch.compile calls them between its graphs.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native_train

__all__ = ["grouped_linear", "linear_act"]


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None,
               activation: str = "none") -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: ``x`` [..., in], ``weight`` [out, in],
    ``bias`` [out], ``residual`` [..., out]; ``activation`` is ``"none"``,
    ``"relu"``, ``"gelu"`` (erf) or ``"silu"``."""
    return _native_train.ext().linear_act(x, weight, bias, residual, activation)


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
    return _native_train.ext().grouped_linear(x, weight, offsets, bias, residual, activation)
