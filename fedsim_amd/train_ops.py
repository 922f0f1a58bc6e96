"""Typed Python wrappers over the libfedtrain C-ABI (include/fedtrain.h): the
dense operators of a training step on the GPU.

Each wrapper checks shapes, types, devices and strides on the host and launches
on the tensors' device, on its current torch stream.  None has a CPU fallback.
``functional`` makes differentiable operators of the products, ``optim`` an
optimizer of the AdamW step.

  product_forward       y = act(x W^T + b) + r, one weight matrix or one a group of rows
  product_grad_input    dx = dz W
  product_grad_weight   dW = dz^T x, db = dz^T 1
  act_backward          dz = dy act'(z)
  adamw_step            AdamW over many tensors, states in 32 or in 8 bits
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _native_train

__all__ = ["ACTIVATIONS", "STATE_BLOCK", "act_backward", "adamw_step", "product_forward",
           "product_grad_input", "product_grad_weight"]

ACTIVATIONS = ("none", "relu", "gelu", "silu")
STATE_BLOCK = 256  # elements of an 8-bit state that share a scale


def product_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    residual: Optional[torch.Tensor] = None, activation: str = "none",
                    offsets: Optional[torch.Tensor] = None, want_z: bool = False
                    ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(y, z) of y = act(z) + residual, z = x weight^T + bias (z only with
    ``want_z``).  ``x`` [N, in], ``weight`` [out, in], ``bias`` [out],
    ``residual`` [N, out]; with ``offsets`` [G + 1] on the device, ``weight``
    [G, out, in] and ``bias`` [G, out], and rows offsets[g] .. offsets[g + 1] of
    ``x`` meet weight[g].  A row in no group gets its residual, or zero."""
    return _native_train.ext().product_forward(x, weight, bias, residual, activation, offsets,
                                               want_z)


def product_grad_input(dz: torch.Tensor, weight: torch.Tensor,
                       offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dx = dz weight ([N, in]), rows in no group zero: the gradient of
    :func:`product_forward`'s x."""
    return _native_train.ext().product_grad_input(dz, weight, offsets)


def product_grad_weight(dz: torch.Tensor, x: torch.Tensor,
                        offsets: Optional[torch.Tensor] = None, want_weight: bool = True,
                        want_bias: bool = False
                        ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dW, db) of :func:`product_forward`: dz^T x ([G,] out, in) and the
    column sums of dz ([G,] out).  A group without rows gets zeros."""
    return _native_train.ext().product_grad_weight(dz, x, offsets, want_weight, want_bias)


def act_backward(dy: torch.Tensor, z: torch.Tensor, activation: str) -> torch.Tensor:
    """dz = dy act'(z), element by element ([N, out]); for ``"relu"`` z may be
    the activation's output."""
    return _native_train.ext().act_backward(dy, z, activation)


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
               exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor],
               exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
               exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None, *, step, lr: float,
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, maximize: bool = False, seed: int = 0,
               first_blocks: Optional[Sequence[int]] = None) -> None:
    """One AdamW step of all ``params``, in place, in one launch for each 62
    tensors::

        m = b1 m + (1 - b1) g            v = b2 v + (1 - b2) g g
        p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    Parameters and gradients are float32, bfloat16 or float16, one type a call;
    the arithmetic is float32 and a 16-bit parameter is rounded once.

    States: ``exp_avgs`` and ``exp_avg_sqs`` float32 like the parameters; or
    float8_e4m3fn and float8_e5m2 codes, with ``exp_avg_scales`` and
    ``exp_avg_sq_scales`` holding a float32 power of two for each 256 elements
    (``STATE_BLOCK``; the last block of a tensor may be short): the state is code
    times scale.  The codes are rounded stochastically, by a hash of ``seed``, the
    step and the element's number (tensors are numbered through in blocks, from
    ``first_blocks[i]`` where given), so a step is the same each time it is run.

    ``step``: 1 for the first step; or an int64 tensor of one element on the
    device, read when the step runs (for a captured graph), or one such tensor
    for each parameter."""
    one = step if isinstance(step, torch.Tensor) else None
    each = step if isinstance(step, (list, tuple)) else None
    _native_train.ext().adamw_step(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales,
                                   exp_avg_sq_scales,
                                   int(step) if one is None and each is None else 0, one, each,
                                   lr, betas[0], betas[1], eps, weight_decay, maximize, seed,
                                   first_blocks)
