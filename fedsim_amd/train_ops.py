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

import contextlib
import ctypes
from typing import Optional, Sequence, Tuple

import torch

from . import _native_train as _nt

__all__ = ["ACTIVATIONS", "STATE_BLOCK", "act_backward", "adamw_step", "product_forward",
           "product_grad_input", "product_grad_weight"]

ACTIVATIONS = {"none": _nt.FEDTRAIN_ACT_NONE, "relu": _nt.FEDTRAIN_ACT_RELU,
               "gelu": _nt.FEDTRAIN_ACT_GELU, "silu": _nt.FEDTRAIN_ACT_SILU}
_DTYPES = {torch.float32: _nt.FEDTRAIN_F32, torch.bfloat16: _nt.FEDTRAIN_BF16,
           torch.float16: _nt.FEDTRAIN_F16}
STATE_BLOCK = 256  # elements of an 8-bit state that share a scale
_MAX = 2 ** 31 - 1


def _on(dev: torch.device):
    """The device a launch needs to be current: a stream handle of 0 is the
    current device's default stream."""
    if dev.index is None or dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _stream_ptr(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _require(t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must live on a HIP device, got {t.device}")
    if like is not None:
        if t.dtype != like.dtype:
            raise TypeError(f"{name} must be {like.dtype} like x, got {t.dtype}")
        if t.device != like.device:
            raise ValueError(f"{name} must live on {like.device}, got {t.device}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with its last dimension's elements next to each other."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _ld(t: torch.Tensor, dim: int = -2) -> int:
    """Elements from one row to the next (anything where there is one row)."""
    if t.shape[dim] > 1:
        return t.stride(dim)
    n = t.shape[-1]
    return n if dim == -2 else n * t.shape[-2]


def _sizes(**named) -> None:
    for name, n in named.items():
        if n > _MAX:
            raise ValueError(f"{name} = {n} is over the largest size, {_MAX}")


def _act(activation: str) -> int:
    try:
        return ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, "
                         f"got {activation!r}") from None


def _groups(w: torch.Tensor, offsets: Optional[torch.Tensor], dev: torch.device):
    """(groups, pointer, is 64 bit) of a grouped product's offsets."""
    if offsets is None:
        return 0, None, 0
    if not isinstance(offsets, torch.Tensor):
        raise TypeError("offsets must be a torch.Tensor")
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"offsets must be int32 or int64, got {offsets.dtype}")
    if offsets.device != dev:
        raise ValueError(f"offsets must live on {dev}, got {offsets.device}")
    G = w.shape[0] if w is not None else offsets.numel() - 1
    if offsets.dim() != 1 or offsets.numel() != G + 1 or G < 1:
        raise ValueError(f"offsets must hold one more value than there are groups ({G}), "
                         f"got shape {tuple(offsets.shape)}")
    if not offsets.is_contiguous():
        raise ValueError("offsets must be contiguous")
    return G, offsets.data_ptr(), int(offsets.dtype == torch.int64)


def _launch(args: "_nt.ProductArgs", dev: torch.device) -> None:
    lib = _nt.load()
    with _on(dev):
        need = lib.fedtrain_product_workspace(ctypes.byref(args))
        work = None
        if need > 0:
            work = torch.empty(need, dtype=torch.uint8, device=dev)
            args.workspace, args.workspace_bytes = work.data_ptr(), need
        rc = lib.fedtrain_product(ctypes.byref(args), _stream_ptr(dev))
    _nt.check(rc, "fedtrain_product")


def product_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    residual: Optional[torch.Tensor] = None, activation: str = "none",
                    offsets: Optional[torch.Tensor] = None, want_z: bool = False
                    ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(y, z) of y = act(z) + residual, z = x weight^T + bias (z only with
    ``want_z``).  ``x`` [N, in], ``weight`` [out, in], ``bias`` [out],
    ``residual`` [N, out]; with ``offsets`` [G + 1] on the device, ``weight``
    [G, out, in] and ``bias`` [G, out], and rows offsets[g] .. offsets[g + 1] of
    ``x`` meet weight[g].  A row in no group gets its residual, or zero."""
    act = _act(activation)
    _require(x, "x")
    _require(weight, "weight", x)
    lead = 1 if offsets is not None else 0
    if x.dim() != 2 or weight.dim() != 2 + lead or weight.shape[-1] != x.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit "
                         f"[N, in] and [{'G, ' * lead}out, in]")
    N, K, M = x.shape[0], x.shape[1], weight.shape[-2]
    _sizes(rows=N, inputs=K, outputs=M)
    G, off, off64 = _groups(weight, offsets, x.device)
    if bias is not None:
        _require(bias, "bias", x)
        if bias.shape != weight.shape[:-1]:
            raise ValueError(f"bias must have shape {tuple(weight.shape[:-1])}, "
                             f"got {tuple(bias.shape)}")
        bias = _rows(bias)
    if residual is not None:
        _require(residual, "residual", x)
        if residual.shape != (N, M):
            raise ValueError(f"residual must have shape {(N, M)}, got {tuple(residual.shape)}")
        residual = _rows(residual)
    x, weight = _rows(x), _rows(weight)
    y = torch.empty((N, M), dtype=x.dtype, device=x.device)
    z = torch.empty_like(y) if want_z else None
    _launch(_nt.ProductArgs(
        dtype=_DTYPES[x.dtype], form=_nt.FEDTRAIN_FORWARD, act=act, groups=G, m=N, n=M, k=K,
        a=x.data_ptr(), lda=_ld(x), b=weight.data_ptr(), ldb=_ld(weight),
        b_group=_ld(weight, -3) if G else 0, c=y.data_ptr(), ldc=M,
        bias=bias.data_ptr() if bias is not None else None,
        bias_group=_ld(bias) if G and bias is not None else 0,
        res=residual.data_ptr() if residual is not None else None,
        ldr=_ld(residual) if residual is not None else 0,
        z=z.data_ptr() if want_z else None, ldz=M, offsets=off, offsets64=off64), x.device)
    return y, z


def product_grad_input(dz: torch.Tensor, weight: torch.Tensor,
                       offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dx = dz weight ([N, in]), rows in no group zero: the gradient of
    :func:`product_forward`'s x."""
    _require(dz, "dz")
    _require(weight, "weight", dz)
    if dz.dim() != 2 or weight.dim() != (3 if offsets is not None else 2) or \
            weight.shape[-2] != dz.shape[1]:
        raise ValueError(f"dz {tuple(dz.shape)} does not fit weight {tuple(weight.shape)}")
    N, M, K = dz.shape[0], dz.shape[1], weight.shape[-1]
    _sizes(rows=N, inputs=K, outputs=M)
    G, off, off64 = _groups(weight, offsets, dz.device)
    dz, weight = _rows(dz), _rows(weight)
    dx = torch.empty((N, K), dtype=dz.dtype, device=dz.device)
    _launch(_nt.ProductArgs(
        dtype=_DTYPES[dz.dtype], form=_nt.FEDTRAIN_GRAD_INPUT, groups=G, m=N, n=K, k=M,
        a=dz.data_ptr(), lda=_ld(dz), b=weight.data_ptr(), ldb=_ld(weight),
        b_group=_ld(weight, -3) if G else 0, c=dx.data_ptr(), ldc=K, offsets=off,
        offsets64=off64), dz.device)
    return dx


def product_grad_weight(dz: torch.Tensor, x: torch.Tensor,
                        offsets: Optional[torch.Tensor] = None, want_weight: bool = True,
                        want_bias: bool = False
                        ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dW, db) of :func:`product_forward`: dz^T x ([G,] out, in) and the
    column sums of dz ([G,] out).  A group without rows gets zeros."""
    _require(x, "x")
    _require(dz, "dz", x)
    if dz.dim() != 2 or x.dim() != 2 or dz.shape[0] != x.shape[0]:
        raise ValueError(f"dz {tuple(dz.shape)} and x {tuple(x.shape)} do not fit")
    N, M, K = dz.shape[0], dz.shape[1], x.shape[1]
    _sizes(rows=N, inputs=K, outputs=M)
    G, off, off64 = _groups(None, offsets, dz.device)
    lead = (G,) if G else ()
    dz, x = _rows(dz), _rows(x)
    dw = torch.empty((*lead, M, K), dtype=x.dtype, device=x.device) if want_weight else None
    db = torch.empty((*lead, M), dtype=x.dtype, device=x.device) if want_bias else None
    if dw is None and db is None:
        return None, None
    _launch(_nt.ProductArgs(
        dtype=_DTYPES[x.dtype], form=_nt.FEDTRAIN_GRAD_WEIGHT, groups=G, m=M,
        n=K if want_weight else 0, k=N, a=dz.data_ptr(), lda=_ld(dz), b=x.data_ptr(), ldb=_ld(x),
        c=dw.data_ptr() if want_weight else None, ldc=K, c_group=M * K,
        colsum=db.data_ptr() if want_bias else None, colsum_group=M, offsets=off,
        offsets64=off64), x.device)
    return dw, db


def act_backward(dy: torch.Tensor, z: torch.Tensor, activation: str) -> torch.Tensor:
    """dz = dy act'(z), element by element ([N, out]); for ``"relu"`` z may be
    the activation's output."""
    act = _act(activation)
    _require(dy, "dy")
    _require(z, "z", dy)
    if dy.dim() != 2 or dy.shape != z.shape:
        raise ValueError(f"dy {tuple(dy.shape)} and z {tuple(z.shape)} must be one [N, out]")
    _sizes(rows=dy.shape[0], outputs=dy.shape[1])
    dy, z = _rows(dy), _rows(z)
    dz = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
    with _on(dy.device):
        rc = _nt.load().fedtrain_act_backward(
            _DTYPES[dy.dtype], act, dy.shape[0], dy.shape[1], dy.data_ptr(), _ld(dy),
            z.data_ptr(), _ld(z), dz.data_ptr(), dz.shape[1], _stream_ptr(dy.device))
    _nt.check(rc, "fedtrain_act_backward")
    return dz


def _same(tensors: Sequence[torch.Tensor], name: str, dtype, dev, sizes) -> None:
    if len(tensors) != len(sizes):
        raise ValueError(f"{name}: {len(tensors)} tensors for {len(sizes)} parameters")
    for i, (t, n) in enumerate(zip(tensors, sizes)):
        if t.dtype != dtype or t.device != dev or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{name}[{i}] must be a contiguous {dtype} tensor of {n} elements "
                             f"on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
               exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor],
               exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
               exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None, *, step, lr: float,
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, maximize: bool = False, seed: int = 0,
               first_blocks: Optional[Sequence[int]] = None) -> None:
    """One AdamW step of all ``params``, in place, in one launch for each 40
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
    device, read when the step runs (for a captured graph)."""
    if not params:
        return
    p0 = params[0]
    _require(p0, "params[0]")
    dt, dev = p0.dtype, p0.device
    sizes = [p.numel() for p in params]
    _same(params, "params", dt, dev, sizes)
    _same(grads, "grads", dt, dev, sizes)
    eight = exp_avg_scales is not None
    if eight != (exp_avg_sq_scales is not None):
        raise ValueError("exp_avg_scales and exp_avg_sq_scales are given together")
    _same(exp_avgs, "exp_avgs", torch.float8_e4m3fn if eight else torch.float32, dev, sizes)
    _same(exp_avg_sqs, "exp_avg_sqs", torch.float8_e5m2 if eight else torch.float32, dev, sizes)
    blocks = [-(-n // STATE_BLOCK) for n in sizes]
    if eight:
        _same(exp_avg_scales, "exp_avg_scales", torch.float32, dev, blocks)
        _same(exp_avg_sq_scales, "exp_avg_sq_scales", torch.float32, dev, blocks)
    b1, b2 = betas
    if not (lr >= 0 and 0 <= b1 < 1 and 0 <= b2 < 1 and eps >= 0 and weight_decay >= 0):
        raise ValueError(f"lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}: "
                         "betas lie in [0, 1), the others are not negative")
    first = first_blocks
    if first is None:
        first, at = [], 0
        for n in blocks:
            first.append(at)
            at += n
    elif len(first) != len(params):
        raise ValueError(f"{len(first)} first_blocks for {len(params)} parameters")
    n = len(params)
    words = [0] * (_nt.ADAMW_WORDS * n)
    for k, ts in enumerate((params, grads, exp_avgs, exp_avg_sqs)):
        words[k::_nt.ADAMW_WORDS] = [t.data_ptr() for t in ts]
    if eight:
        words[4::_nt.ADAMW_WORDS] = [t.data_ptr() for t in exp_avg_scales]
        words[5::_nt.ADAMW_WORDS] = [t.data_ptr() for t in exp_avg_sq_scales]
    words[6::_nt.ADAMW_WORDS] = sizes
    words[7::_nt.ADAMW_WORDS] = first
    table = (ctypes.c_int64 * len(words))(*words)
    work = None
    s = _nt.AdamWScalars(lr=lr, beta1=b1, beta2=b2, eps=eps, weight_decay=weight_decay,
                         seed=seed & 0xFFFFFFFF, maximize=int(bool(maximize)))
    with _on(dev):
        if isinstance(step, torch.Tensor):
            if step.dtype != torch.int64 or step.device != dev or step.numel() != 1:
                raise ValueError(f"a step on the device must be one int64 on {dev}")
            work = torch.empty(4, dtype=torch.float32, device=dev)
            s.device_step, s.workspace = step.data_ptr(), work.data_ptr()
        else:
            if step < 1:
                raise ValueError(f"steps are counted from 1, got {step}")
            s.step = int(step)
        rc = _nt.load().fedtrain_adamw(_DTYPES[dt], 8 if eight else 32, n,
                                       ctypes.cast(table, ctypes.c_void_p), ctypes.byref(s),
                                       _stream_ptr(dev))
    _nt.check(rc, "fedtrain_adamw")
