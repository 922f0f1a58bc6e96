"""What the dense training operators refuse, on the CPU: the Python checks and
the C entries' own, before any device work."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from conftest import REPO

HEADER = os.path.join(REPO, "include", "fedtrain.h")
LIB = os.path.join(REPO, "fedsim_amd", "libfedtrain.so")
E = -22


@pytest.fixture(scope="module")
def lib():
    from fedsim_amd import _native_train

    return _native_train.load()


def _functions():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(fedtrain_[a-z_]+)\s*\(", text)))


def test_library_exports_what_the_header_declares(lib):
    from fedsim_amd import _native_train

    out = subprocess.check_output(["nm", "-D", "--defined-only", LIB], text=True)
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert set(_functions()) == set(_native_train.exported_symbols())
    assert set(_functions()) <= exported
    text = open(HEADER).read()
    for name, value in re.findall(r"#define\s+(FEDTRAIN_[A-Z0-9_]+)\s+\(?(-?\d+)\)?", text):
        mirror = "ABI_VERSION" if name == "FEDTRAIN_ABI_VERSION" else name
        assert getattr(_native_train, mirror) == int(value), name


def _args(**kw):
    from fedsim_amd import _native_train as nt

    d = dict(dtype=0, form=0, m=4, n=4, k=4, a=64, lda=4, b=64, ldb=4, c=64, ldc=4)
    d.update(kw)
    return nt.ProductArgs(**d)


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(form=3), dict(act=4), dict(act=-1), dict(m=-1),
    dict(n=-1), dict(k=-1), dict(m=1 << 31), dict(n=1 << 31), dict(k=1 << 31), dict(groups=-1),
    dict(groups=2), dict(a=None), dict(b=None), dict(c=None), dict(a=66), dict(b=65), dict(c=62),
    dict(ldc=3), dict(lda=-4), dict(ldb=-4), dict(z=64, ldz=3), dict(bias=66), dict(res=66),
    dict(colsum=64), dict(form=1, act=1), dict(form=1, bias=64), dict(form=1, res=64),
    dict(form=2, z=64, ldz=4), dict(form=2, c=None), dict(groups=2, offsets=66),
    dict(groups=2, offsets=68, offsets64=1), dict(form=2, groups=2, offsets=64, c_group=15),
    dict(form=2, groups=2, offsets=64, c_group=16, colsum=64, colsum_group=3),
    dict(groups=2147483647, offsets=64),
], ids=str)
def test_product_refusals(lib, bad):
    a = _args(**bad)
    assert lib.fedtrain_product(ctypes.byref(a), None) == E
    assert lib.fedtrain_product_workspace(ctypes.byref(a)) == E


def test_product_without_work(lib):
    assert lib.fedtrain_product(None, None) == E
    for kw in (dict(m=0), dict(n=0), dict(m=0, a=None, b=None, c=None),
               dict(form=2, m=0, a=None, b=None, c=None)):
        assert lib.fedtrain_product(ctypes.byref(_args(**kw)), None) == 0


def _plan(lib, **kw):
    got = [ctypes.c_int() for _ in range(3)]
    assert lib.fedtrain_product_plan(ctypes.byref(_args(**kw)),
                                     *(ctypes.byref(g) for g in got)) == 0
    return tuple(g.value for g in got)


# (dtype, aligned, form, sizes) -> the tile and whether k is taken in parts
PLANS = [
    (1, True, 0, (4001, 4008, 3976), (256, 256), False),
    (2, True, 1, (4001, 3976, 4008), (256, 256), False),
    (1, True, 2, (4008, 3976, 4001), (256, 256), False),
    (2, True, 0, (2048, 2048, 520), (128, 128), False),
    (1, True, 1, (4000, 520, 4008), (128, 128), True),
    (1, True, 2, (1024, 2304, 264), (128, 128), False),
    (1, True, 0, (300, 520, 136), (64, 64), False),
    (1, True, 1, (64, 200, 4096), (64, 64), True),
    (2, False, 0, (2049, 2047, 517), (128, 128), False),
    (1, False, 2, (300, 261, 135), (64, 64), False),
    (1, False, 0, (40, 33, 5001), (64, 64), True),
    (0, True, 0, (3000, 2500, 300), (128, 128), False),
    (0, False, 1, (700, 900, 100), (64, 128), False),
    (0, True, 2, (500, 100, 9000), (64, 128), True),
    (0, False, 0, (4, 300, 1000), (4, 1), False),
    (1, True, 0, (1, 4096, 4096), (1, 1), False),
]


@pytest.mark.parametrize("dtype,aligned,form,mnk,tile,parts", PLANS, ids=str)
def test_plans(lib, dtype, aligned, form, mnk, tile, parts):
    """Which kernel takes what: each of them is taken somewhere."""
    m, n, k = mnk
    lda, ldb = (k, k) if form == 0 else (k, n) if form == 1 else (m, n)
    got = _plan(lib, dtype=dtype, form=form, m=m, n=n, k=k, lda=lda, ldb=ldb, ldc=n,
                a=64 if aligned else 68)
    assert got[:2] == tile and (got[2] > 1) == parts, got


def test_plan_refusals(lib):
    i = ctypes.c_int()
    r = ctypes.byref(i)
    assert lib.fedtrain_product_plan(ctypes.byref(_args(dtype=9)), r, r, r) == E
    assert lib.fedtrain_product_plan(ctypes.byref(_args()), None, r, r) == E
    assert lib.fedtrain_product_plan(None, r, r, r) == E


def test_more_tiles_than_a_launch_holds(lib):
    big = (1 << 31) - 1
    for kw in (dict(m=big, n=1, k=1), dict(m=big, n=2, k=1, form=1, lda=1),
               dict(m=big, n=2, k=1, form=2, ldc=4), dict(m=1, n=big, k=1, dtype=1, ldc=big)):
        a = _args(**kw)
        assert lib.fedtrain_product_workspace(ctypes.byref(a)) >= 0
        assert lib.fedtrain_product(ctypes.byref(a), None) == E
    assert lib.fedtrain_act_backward(1, 1, 1 << 18, 1 << 18, 64, 1 << 18, 64, 1 << 18, 64, 1 << 18,
                                     None) == E


def test_act_backward_refusals(lib):
    f = lib.fedtrain_act_backward
    ok = [0, 1, 2, 4, 64, 4, 64, 4, 64, 4, None]
    for i, v in ((0, 3), (1, 4), (1, -1), (2, -1), (3, -1), (2, 1 << 31), (4, None), (6, None),
                 (8, None), (4, 66), (6, 66), (8, 66), (5, -1), (7, -1), (9, 3)):
        bad = list(ok)
        bad[i] = v
        assert f(*bad) == E, (i, v)
    assert f(0, 1, 0, 4, None, 0, None, 0, None, 0, None) == 0


def test_adamw_refusals(lib):
    from fedsim_amd import _native_train as nt

    def call(dtype=0, bits=32, count=1, words=None, none=False, **kw):
        s = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, step=1)
        s.update(kw)
        w = dict(p=64, g=64, m=64, v=64, ms=64, vs=64, n=10, b0=0)
        w.update(words or {})
        table = (ctypes.c_int64 * 8)(*w.values())
        return lib.fedtrain_adamw(dtype, bits, count,
                                  None if none else ctypes.cast(table, ctypes.c_void_p),
                                  ctypes.byref(nt.AdamWScalars(**s)), None)

    assert call(words=dict(n=0)) == 0
    assert call(count=0, none=True) == 0
    bad = [dict(dtype=3), dict(dtype=-1), dict(bits=16), dict(count=-1), dict(none=True),
           dict(step=0), dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(lr=-1.0),
           dict(eps=-1.0), dict(weight_decay=-1.0), dict(lr=float("nan")),
           dict(device_step=64), dict(device_step=64, workspace=66)]
    bad += [dict(words={k: 0}) for k in ("p", "g", "m", "v")]
    bad += [dict(words={k: 66}) for k in ("p", "g", "m", "v")]
    bad += [dict(bits=8, words={k: v}) for k in ("ms", "vs") for v in (0, 66)]
    bad += [dict(words=dict(n=-1)), dict(words=dict(b0=-1)), dict(words=dict(n=1 << 50))]
    for kw in bad:
        assert call(**kw) == E, kw
    assert lib.fedtrain_adamw(0, 32, 0, None, None, None) == E


def test_functions_refuse_host_tensors():
    from fedsim_amd import train_ops
    from fedsim_amd.functional import grouped_linear, linear_act
    from fedsim_amd.optim import AdamW

    x, w = torch.zeros(3, 4), torch.zeros(5, 4)
    with pytest.raises(ValueError, match="HIP device"):
        linear_act(x, w)
    with pytest.raises(ValueError, match="HIP device"):
        grouped_linear(x, w[None], torch.tensor([0, 3]))
    with pytest.raises(ValueError, match="HIP device"):
        train_ops.act_backward(x, x, "relu")
    with pytest.raises(ValueError, match="HIP device"):
        train_ops.product_grad_weight(x, x)
    with pytest.raises(ValueError, match="HIP device"):
        train_ops.product_grad_input(x, w)
    with pytest.raises(TypeError):
        linear_act(x.double(), w.double())
    with pytest.raises(TypeError):
        linear_act([1.0], w)
    with pytest.raises(TypeError):
        grouped_linear(x, w[None], None)
    with pytest.raises(ValueError, match="activation"):
        train_ops.product_forward(x, w, activation="tanh")
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    opt = AdamW([p])
    with pytest.raises(ValueError, match="HIP device"):
        opt.step()
    with pytest.raises(ValueError, match="HIP device"):
        train_ops.adamw_step([p], [p], [p], [p], step=1, lr=1e-3)


@pytest.mark.parametrize("kw", [dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
                                dict(eps=-1e-8), dict(weight_decay=-1.0), dict(state_bits=16)],
                         ids=str)
def test_optimizer_refuses_arguments(kw):
    from fedsim_amd.optim import AdamW

    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(4))], **kw)


@pytest.mark.gpu
def test_functions_refuse_what_does_not_fit():
    from fedsim_amd import train_ops
    from fedsim_amd.functional import grouped_linear, linear_act

    def t(*s, dtype=torch.float32):
        return torch.zeros(*s, dtype=dtype, device="cuda")

    bf = torch.bfloat16
    for bad in (lambda: linear_act(t(3, 4), t(5, 6)), lambda: linear_act(t(3, 4), t(4)),
                lambda: linear_act(t(3, 4), t(5, 4), t(4)),
                lambda: linear_act(t(3, 4), t(5, 4), None, t(3, 4)),
                lambda: linear_act(t(3, 4), t(5, 4), None, t(2, 5)),
                lambda: linear_act(t(3, 4), t(5, 4), activation="tanh"),
                lambda: grouped_linear(t(3, 4), t(5, 4), torch.tensor([0, 3], device="cuda")),
                lambda: grouped_linear(t(3, 4), t(2, 5, 4), torch.tensor([0, 3], device="cuda")),
                lambda: grouped_linear(t(3, 4), t(1, 5, 4), torch.tensor([0, 3])),
                lambda: grouped_linear(t(3, 4), t(1, 5, 4), torch.tensor([[0], [3]],
                                                                         device="cuda")),
                lambda: grouped_linear(t(3, 4), t(1, 5, 4),
                                       torch.tensor([0, 1, 3, 3], device="cuda")[::2]),
                lambda: grouped_linear(t(3, 4), t(0, 5, 4), torch.tensor([0], device="cuda")),
                lambda: grouped_linear(t(3, 4), t(1, 5, 4), torch.tensor([0, 3], device="cuda"),
                                       t(5)),
                lambda: train_ops.act_backward(t(3, 4), t(4, 3), "relu"),
                lambda: train_ops.product_grad_weight(t(3, 4), t(4, 3)),
                lambda: train_ops.product_grad_input(t(3, 4), t(5, 4))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: linear_act(t(3, 4), t(5, 4, dtype=bf)),
                lambda: linear_act(t(3, 4), t(5, 4), t(5, dtype=bf)),
                lambda: linear_act(t(3, 4), t(5, 4), None, t(3, 5, dtype=bf)),
                lambda: grouped_linear(t(3, 4), t(1, 5, 4), torch.tensor([0., 3.],
                                                                         device="cuda"))):
        with pytest.raises(TypeError):
            bad()
    f8, f8v = torch.float8_e4m3fn, torch.float8_e5m2
    ok = dict(step=1, lr=1e-3)
    p, s = t(300), t(2)
    for bad in (lambda: train_ops.adamw_step([p], [], [p], [p], **ok),
                lambda: train_ops.adamw_step([p], [t(299)], [p], [p], **ok),
                lambda: train_ops.adamw_step([p], [t(300, dtype=bf)], [p], [p], **ok),
                lambda: train_ops.adamw_step([p], [p], [t(600)[::2]], [p], **ok),
                lambda: train_ops.adamw_step([p], [p], [t(300, dtype=bf)], [p], **ok),
                lambda: train_ops.adamw_step([p], [p], [p], [p], [s], [s], **ok),
                lambda: train_ops.adamw_step([p], [p], [p.to(f8)], [p.to(f8v)], **ok),
                lambda: train_ops.adamw_step([p], [p], [p.to(f8)], [p.to(f8v)], [s], **ok),
                lambda: train_ops.adamw_step([p], [p], [p.to(f8)], [p.to(f8v)], [t(1)], [s], **ok),
                lambda: train_ops.adamw_step([p], [p], [p], [p], step=0, lr=1e-3),
                lambda: train_ops.adamw_step([p], [p], [p], [p], step=t(1), lr=1e-3),
                lambda: train_ops.adamw_step([p], [p], [p], [p], step=1, lr=1e-3,
                                             betas=(0.9, 1.0)),
                lambda: train_ops.adamw_step([p, p], [p, p], [p, p], [p, p], **ok),
                lambda: train_ops.adamw_step([p[:200], p[100:]], [p[:200], p[100:]],
                                             [t(200), t(200)], [t(200), t(200)], **ok),
                lambda: train_ops.adamw_step([t(2), t(2)], [s, s], [s, s], [t(2), t(2)], **ok),
                lambda: train_ops.adamw_step([p], [p], [p], [p], first_blocks=[], **ok)):
        with pytest.raises(ValueError):
            bad()
    assert train_ops.adamw_step([], [], [], [], **ok) is None
