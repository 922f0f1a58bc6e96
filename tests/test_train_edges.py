"""The training operators' edges that need no device: C arguments, tracing, what
the compiler spilled."""
import ctypes
import re
import subprocess

import pytest
import torch

from test_train_isa import NM, _instructions, objects  # noqa: F401  (one a fixture)

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


def test_act_backward_sums_refusals():
    from fedsim_amd import _native_train as nt

    lib = nt.load()

    def args(**kw):
        d = dict(dtype=1, act=2, rows=10, cols=4, dy=64, lddy=4, z=64, ldz=4, dz=64, lddz=4,
                 colsum=64)
        d.update(kw)
        return ctypes.byref(nt.ActArgs(**d))

    size = lib.fedtrain_act_backward_sums_workspace
    assert size(args()) == size(args(rows=32)) == size(args(rows=0)) == 0
    assert size(args(rows=33)) == 2 * 4 * 4
    grouped = dict(groups=3, offsets=64, colsum_group=4)
    assert size(args(**grouped)) == 5 * 4 * 4
    assert size(args(rows=5000, **grouped)) == (5000 // 32 + 5) * 4 * 4
    assert size(args(rows=1 << 20)) == 256 * 4 * 4  # no more parts than that
    assert size(args(rows=8192, cols=16384, lddz=16384)) == 128 * 16384 * 4
    call = lib.fedtrain_act_backward_sums
    assert call(args(cols=0), None) == call(args(cols=0, dy=None, z=None, dz=None, colsum=None),
                                            None) == 0
    assert call(None, None) == size(None) == E
    for bad in (dict(dtype=0), dict(dtype=3), dict(act=4), dict(act=-1), dict(groups=-1),
                dict(groups=2147483647, offsets=64), dict(rows=-1), dict(cols=-1),
                dict(rows=1 << 31), dict(cols=1 << 31), dict(dy=None), dict(z=None), dict(dz=None),
                dict(colsum=None), dict(dy=65), dict(z=65), dict(dz=65), dict(colsum=65),
                dict(lddy=-1), dict(ldz=-1), dict(lddz=3), dict(groups=2),
                dict(groups=2, offsets=66, colsum_group=4),
                dict(groups=2, offsets=68, offsets64=1, colsum_group=4),
                dict(groups=2, offsets=64, colsum_group=3)):
        assert call(args(**bad), None) == E and size(args(**bad)) == E, bad
    for bad in (dict(rows=33), dict(**grouped), dict(rows=33, workspace=68, workspace_bytes=32),
                dict(rows=33, workspace=64, workspace_bytes=31)):
        assert call(args(**bad), None) == E and size(args(**bad)) > 0, bad
    # more workgroups than a launch holds
    wide = args(rows=1 << 20, cols=(1 << 31) - 1, lddz=1 << 31)
    assert size(wide) == 0 and call(wide, None) == E


def _calls():
    """(name, function of two tensors, its arguments' shapes)."""
    from fedsim_amd import train_ops
    from fedsim_amd.functional import grouped_linear, linear_act

    off = torch.tensor([0, 3])
    return [
        ("linear_act", lambda x, w: linear_act(x, w), (3, 4), (5, 4)),
        ("grouped_linear", lambda x, w: grouped_linear(x, w[None], off), (3, 4), (5, 4)),
        ("forward", lambda x, w: train_ops.product_forward(x, w)[0], (3, 4), (5, 4)),
        ("grad_input", lambda d, w: train_ops.product_grad_input(d, w), (3, 5), (5, 4)),
        ("grad_weight", lambda d, x: train_ops.product_grad_weight(d, x)[0], (3, 5), (3, 4)),
        ("act_backward", lambda d, z: train_ops.act_backward(d, z, "relu"), (3, 5), (3, 5)),
        ("adamw_step", lambda p, g: train_ops.adamw_step(
            [p], [g], [g * 0], [g * 0], step=1, lr=1e-3), (8,), (8,)),
    ]


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("k", range(7))
def test_tracing_is_refused(k):
    """A recorded graph would hold the allocation of the results and not what
    fills them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    name, f, a, b = _calls()[k]
    x, y = torch.randn(a), torch.randn(b)

    class Module(torch.nn.Module):
        def forward(self, x, y):
            return f(x, y)

    def fake():
        with FakeTensorMode():
            f(torch.empty(a, device="cuda"), torch.empty(b, device="cuda"))

    for trace in (lambda: torch.jit.trace(f, (x, y)), lambda: make_fx(f)(x, y),
                  lambda: make_fx(f, tracing_mode="fake")(x, y),
                  lambda: make_fx(f, tracing_mode="symbolic")(x, y),
                  lambda: make_fx(f, pre_dispatch=True)(x, y),
                  lambda: torch.export.export(Module(), (x, y), strict=False), fake):
        with pytest.raises(NotImplementedError, match="traced"):
            trace()
    with pytest.raises(ValueError, match="HIP device"):  # and nothing of it stays behind
        f(x, y)


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_transforms_raise_and_compile_breaks_its_graph():
    """torch.func's wrapped tensors have no memory to read; torch.compile calls
    the operators outside its graphs."""
    from torch.utils.flop_counter import FlopCounterMode

    from fedsim_amd.functional import linear_act

    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn(3, 4, generator=gen).cuda(), torch.randn(5, 4, generator=gen).cuda()
    for bad in (lambda: torch.vmap(lambda a: linear_act(a, w))(torch.stack([x, x])),
                lambda: torch.func.grad(lambda a: linear_act(a, w).sum())(x),
                lambda: torch.func.functionalize(lambda a: linear_act(a, w))(x)):
        with pytest.raises(RuntimeError):
            bad()
    want = linear_act(x, w, activation="gelu")
    got = torch.compile(lambda a: linear_act(a * 1, w, activation="gelu") * 1, backend="eager")(x)
    assert torch.equal(got, want)
    with FlopCounterMode(display=False):  # a mode that looks on is no tracer
        assert torch.equal(linear_act(x, w, activation="gelu"), want)


def test_m0_belongs_to_the_direct_loads(objects):
    """The loads to LDS set m0 in assembly, and the compiler takes no such clobber
    (m0 is reserved): so nothing it emits may name m0 itself, or read it unnamed."""
    sets = loads = 0
    for co in objects:
        last = []
        for _, op, args in _instructions(co):
            if "m0" in args.replace(",", " ").split():
                assert op == "s_mov_b32" and args.startswith("m0, s"), (op, args)
                sets += 1
            # what reads m0 without naming it
            assert not op.startswith(("v_movrel", "s_movrel", "s_set_gpr_idx", "v_interp",
                                      "s_sendmsg", "ds_gws", "s_ttracedata")), op
            if " lds" in args or op.startswith("global_load_lds"):
                loads += 1
                assert op.startswith("buffer_load") and [o for o, _ in last[-2:]] == \
                    ["s_mov_b32", "s_nop"] and last[-2][1].startswith("m0"), last
            last = (last + [(op, args)])[-2:]
    assert sets == loads > 1000


def test_spilled_registers(objects):
    """No vector register is spilled; of scalars the widest grad weight keeps five in a
    vector register's lanes."""
    seen = 0
    for co in objects:
        notes = subprocess.check_output([NM, "--notes", co], text=True)
        for key, most in ((".vgpr_spill_count", 0), (".sgpr_spill_count", 8)):
            counts = [int(n) for n in re.findall(re.escape(key) + r":\s+(\d+)", notes)]
            assert counts and max(counts) <= most, (key, counts)
            seen += len(counts)
    assert seen > 100
