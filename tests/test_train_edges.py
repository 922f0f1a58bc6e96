"""The training operators' edges that need no device: C arguments, tracing, what
the compiler spilled."""
import ctypes

import pytest
import torch

E = -22


def test_counts_on_the_device_are_checked():
    """One address for each tensor with elements, 8-byte aligned, and a workspace."""
    from fedsim_amd import _native_train as nt

    lib = nt.load()

    def call(steps, count=2, n=(10, 10), workspace=64):
        words = [[64, 64, 64, 64, 0, 0, k, 0] for k in n[:count]]
        table = (ctypes.c_int64 * (8 * count))(*[w for ws in words for w in ws])
        at = (ctypes.c_int64 * count)(*steps)
        s = nt.AdamWScalars(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=0,
                            workspace=workspace,
                            device_steps=ctypes.cast(at, ctypes.c_void_p))
        return lib.fedtrain_adamw(0, 32, count, ctypes.cast(table, ctypes.c_void_p),
                                  ctypes.byref(s), None)

    assert call((64, 64), n=(0, 0)) == 0 and call((0, 0), n=(0, 0)) == 0
    for kw in (dict(steps=(64, 0)), dict(steps=(0, 64)), dict(steps=(64, 68)),
               dict(steps=(64, 64), workspace=None), dict(steps=(64, 64), workspace=66)):
        assert call(**kw) == E, kw
