"""Loader for libfedtrain.so, the dense training operators' C-ABI
(include/fedtrain.h), and for ``_fedtrain``, the module that calls it on torch
tensors (csrc/fedtrain_binding.cpp).  As with libfedagg (``_native``), torch's
HIP runtime is mapped first and there is no fallback: a missing library raises.
"""
from __future__ import annotations

import ctypes
import importlib
import os
import threading

import torch  # noqa: F401  (must precede the dlopen below)

from ._native import FedAggError, _hip_runtimes_mapped

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libfedtrain.so")

# Must match include/fedtrain.h
ABI_VERSION = 3
FEDTRAIN_EINVAL = -22
FEDTRAIN_F32, FEDTRAIN_BF16, FEDTRAIN_F16 = 0, 1, 2
FEDTRAIN_ACT_NONE, FEDTRAIN_ACT_RELU, FEDTRAIN_ACT_GELU, FEDTRAIN_ACT_SILU = 0, 1, 2, 3
FEDTRAIN_FORWARD, FEDTRAIN_GRAD_INPUT, FEDTRAIN_GRAD_WEIGHT = 0, 1, 2


class ProductArgs(ctypes.Structure):
    """struct fedtrain_product_args (include/fedtrain.h)."""

    _fields_ = ([(n, ctypes.c_int32) for n in ("dtype", "form", "act", "groups")]
                + [(n, ctypes.c_int64) for n in ("m", "n", "k")]
                + [("a", ctypes.c_void_p), ("lda", ctypes.c_int64),
                   ("b", ctypes.c_void_p), ("ldb", ctypes.c_int64), ("b_group", ctypes.c_int64),
                   ("c", ctypes.c_void_p), ("ldc", ctypes.c_int64), ("c_group", ctypes.c_int64),
                   ("bias", ctypes.c_void_p), ("bias_group", ctypes.c_int64),
                   ("res", ctypes.c_void_p), ("ldr", ctypes.c_int64),
                   ("z", ctypes.c_void_p), ("ldz", ctypes.c_int64),
                   ("colsum", ctypes.c_void_p), ("colsum_group", ctypes.c_int64),
                   ("offsets", ctypes.c_void_p), ("offsets64", ctypes.c_int32),
                   ("reserved", ctypes.c_int32),
                   ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64)])


class ActArgs(ctypes.Structure):
    """struct fedtrain_act_args (include/fedtrain.h)."""

    _fields_ = ([(n, ctypes.c_int32) for n in ("dtype", "act", "groups", "offsets64")]
                + [("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
                   ("dy", ctypes.c_void_p), ("lddy", ctypes.c_int64),
                   ("z", ctypes.c_void_p), ("ldz", ctypes.c_int64),
                   ("dz", ctypes.c_void_p), ("lddz", ctypes.c_int64),
                   ("colsum", ctypes.c_void_p), ("colsum_group", ctypes.c_int64),
                   ("offsets", ctypes.c_void_p),
                   ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64)])


class AdamWScalars(ctypes.Structure):
    """struct fedtrain_adamw_scalars (include/fedtrain.h)."""

    _fields_ = ([(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay")]
                + [("step", ctypes.c_int64), ("seed", ctypes.c_uint32),
                   ("maximize", ctypes.c_int32), ("device_step", ctypes.c_void_p),
                   ("workspace", ctypes.c_void_p), ("device_steps", ctypes.c_void_p)])


SIGNATURES = {
    "fedtrain_abi_version": (ctypes.c_int, []),
    "fedtrain_strerror": (ctypes.c_char_p, [ctypes.c_int]),
    "fedtrain_product_workspace": (ctypes.c_int64, [ctypes.POINTER(ProductArgs)]),
    "fedtrain_product_plan": (
        ctypes.c_int,
        [ctypes.POINTER(ProductArgs)] + [ctypes.POINTER(ctypes.c_int)] * 3,
    ),
    "fedtrain_product": (ctypes.c_int, [ctypes.POINTER(ProductArgs), ctypes.c_void_p]),
    "fedtrain_act_backward": (
        ctypes.c_int,
        [ctypes.c_int, ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p,
         ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64,
         ctypes.c_void_p],
    ),
    "fedtrain_act_backward_sums_workspace": (ctypes.c_int64, [ctypes.POINTER(ActArgs)]),
    "fedtrain_act_backward_sums": (ctypes.c_int, [ctypes.POINTER(ActArgs), ctypes.c_void_p]),
    "fedtrain_adamw": (
        ctypes.c_int,
        [ctypes.c_int, ctypes.c_int, ctypes.c_int64, ctypes.c_void_p,
         ctypes.POINTER(AdamWScalars), ctypes.c_void_p],
    ),
}

_lock = threading.Lock()
_lib = None
_ext = None


def ext():
    """The module ``_fedtrain`` (loaded once); raise if unavailable."""
    global _ext
    if _ext is None:
        load()
        try:
            _ext = importlib.import_module("._fedtrain", __package__)
        except ImportError as e:
            raise FedAggError(f"fedsim_amd._fedtrain cannot be loaded ({e}): build it with "
                              "`python -c 'import __graft_entry__ as g; g.build()'`") from e
    return _ext


def load():
    """Load (once) and return the ctypes handle; raise if unavailable."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            raise FedAggError(
                f"{LIB_PATH} not found: build it with `python -c "
                f"'import __graft_entry__ as g; g.build()'` (no CPU fallback exists)"
            )
        lib = ctypes.CDLL(LIB_PATH)
        lib.fedtrain_abi_version.restype = ctypes.c_int
        lib.fedtrain_abi_version.argtypes = []
        built = lib.fedtrain_abi_version()
        if built != ABI_VERSION:
            raise FedAggError(f"{LIB_PATH} has ABI version {built}, this package needs "
                              f"{ABI_VERSION}; rebuild the library")
        for name, (res, args) in SIGNATURES.items():
            try:
                fn = getattr(lib, name)
            except AttributeError:
                raise FedAggError(f"{LIB_PATH} does not export {name}; rebuild the library") \
                    from None
            fn.restype = res
            fn.argtypes = args
        runtimes = _hip_runtimes_mapped()
        if len(runtimes) > 1:
            raise FedAggError("two HIP runtimes are mapped (%s); import torch before fedsim_amd"
                              % sorted(runtimes))
        _lib = lib
        return lib


def exported_symbols():
    """Names of the C-ABI entry points (the ones include/fedtrain.h declares)."""
    return list(SIGNATURES)
