"""Optimizers whose step is one kernel (train_ops.adamw_step)."""
from __future__ import annotations

from typing import Iterable, Tuple

import torch

from . import train_ops

__all__ = ["AdamW"]

_STATES = {32: (torch.float32, torch.float32), 8: (torch.float8_e4m3fn, torch.float8_e5m2)}
_NAMES = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's step (decoupled weight decay, bias correction) over
    all parameters at once, on a HIP device.  An ``optimizer_def`` of it serves
    the clients' local training and the server step alike.

    ``state_bits=8`` holds the moments in e4m3 and e5m2 codes with a power of
    two for each 256 elements: 2 bytes an element instead of 8.  The codes are
    rounded stochastically from ``seed``, the step's number and the element's.

    Each parameter counts its own steps, as a parameter without a gradient sits a
    step out: on the host, or with ``capturable=True`` on the device, so that a
    captured graph of ``step()`` goes on counting when it is replayed.  Capture
    after an eager step, which makes the states; without ``capturable`` a capture
    raises.

    Parameters are contiguous float32, bfloat16 or float16 tensors; a 16-bit
    parameter is rounded to nearest each step.  The step of a captured graph
    uses the learning rate it was captured with."""

    def __init__(self, params: Iterable, lr: float = 1e-3,
                 betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, seed: int = 0,
                 maximize: bool = False, capturable: bool = False):
        if state_bits not in _STATES:
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not (lr >= 0 and 0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0
                and weight_decay >= 0):
            raise ValueError(f"lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}: "
                             "betas lie in [0, 1), the others are not negative")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps,
                                      weight_decay=weight_decay, state_bits=state_bits, seed=seed,
                                      maximize=maximize, capturable=capturable))

    def _init_state(self, p, group, st):
        m, v = _STATES[group["state_bits"]]
        st["exp_avg"] = torch.zeros(p.shape, dtype=m, device=p.device)
        st["exp_avg_sq"] = torch.zeros(p.shape, dtype=v, device=p.device)
        if group["state_bits"] == 8:
            blocks = -(-p.numel() // train_ops.STATE_BLOCK)
            st["exp_avg_scale"] = torch.ones(blocks, dtype=torch.float32, device=p.device)
            st["exp_avg_sq_scale"] = torch.ones(blocks, dtype=torch.float32, device=p.device)
        st["step"] = 0

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        block = 0
        for group in self.param_groups:
            todo = {}  # (type, device, step) -> parameters of one call
            for p in group["params"]:
                first, block = block, block - (-p.numel() // train_ops.STATE_BLOCK)
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                if p.device.type != "cuda" or not p.is_contiguous():
                    raise ValueError("a parameter must be a contiguous tensor on a HIP device, "
                                     f"got strides {p.stride()} on {p.device}")
                st = self.state[p]
                capturing = torch.cuda.is_current_stream_capturing()
                if not st:
                    if capturing:
                        raise RuntimeError("take a step before capturing one: the first makes "
                                           "the states")
                    self._init_state(p, group, st)
                if group["capturable"]:
                    if not isinstance(st["step"], torch.Tensor):
                        if capturing:  # a replay would start again
                            raise RuntimeError("take a step before capturing one: the first "
                                               "puts the count on the device")
                        st["step"] = torch.full((1,), int(st["step"]), dtype=torch.int64,
                                                device=p.device)
                    key = (p.dtype, p.device, None)
                elif capturing:
                    raise RuntimeError("AdamW counts its steps on the host: a captured graph "
                                       "needs capturable=True")
                else:
                    key = (p.dtype, p.device, int(st["step"]) + 1)
                todo.setdefault(key, []).append((p, st, first))
            for (_, _, n), items in todo.items():
                counts = None
                if n is None:
                    counts = [st["step"] for _, st, _ in items]
                    torch._foreach_add_(counts, 1)
                eight = group["state_bits"] == 8
                try:
                    train_ops.adamw_step(
                        [p for p, _, _ in items], [p.grad.contiguous() for p, _, _ in items],
                        [st["exp_avg"] for _, st, _ in items],
                        [st["exp_avg_sq"] for _, st, _ in items],
                        [st["exp_avg_scale"] for _, st, _ in items] if eight else None,
                        [st["exp_avg_sq_scale"] for _, st, _ in items] if eight else None,
                        step=n if counts is None else counts, lr=float(group["lr"]),
                        betas=group["betas"], eps=group["eps"],
                        weight_decay=group["weight_decay"], maximize=group["maximize"],
                        seed=group["seed"], first_blocks=[f for _, _, f in items])
                except Exception:  # a step that was not taken is not counted
                    if counts is not None:
                        torch._foreach_sub_(counts, 1)
                    raise
                if counts is None:
                    for _, st, _ in items:
                        st["step"] = n
        return loss

    def load_state_dict(self, state_dict):
        """torch's, with the states in their own types: torch would cast them
        to the parameters'.  As there, the groups' options are the saved ones,
        ``state_bits`` among them; those that a state of torch.optim.AdamW lacks
        stay as they are."""
        saved = state_dict["param_groups"]
        lacking = [{k: v for k, v in mine.items() if k not in g}
                   for mine, g in zip(self.param_groups, saved)]
        for mine, g in zip(lacking, saved):
            for name, only in (("amsgrad", False), ("decoupled_weight_decay", True)):
                if g.get(name, only) != only:
                    raise ValueError(f"AdamW has no {name}={g[name]}")
            bits = g.get("state_bits", mine.get("state_bits"))
            for i in g["params"]:
                held = state_dict["state"].get(i, {}).get("exp_avg")
                if held is not None and held.dtype != _STATES[bits][0]:
                    raise ValueError(f"a {held.dtype} exp_avg does not fit state_bits={bits}")
        super().load_state_dict(state_dict)
        for g, mine in zip(self.param_groups, lacking):
            g.update(mine)
        ids = [i for g in saved for i in g["params"]]
        ps = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, ps):
            given = state_dict["state"].get(i)
            if not given:
                continue
            st = self.state[p]
            for name in _NAMES:
                if name in given:
                    st[name] = given[name].detach().to(p.device, copy=True)
            if isinstance(given["step"], torch.Tensor):
                st["step"] = int(given["step"])
