"""linear_act and grouped_linear against their definitions in 64 bits
(train_reference.py, with bounds for every element)."""
import pytest
import torch

import train_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "gelu", "silu"]
DEV = "cuda"


def _randn(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * scale).to(dtype)


def _case(N, i, o, dtype, seed, groups=None, bias=True, residual=True):
    gen = torch.Generator().manual_seed(seed)
    lead = () if groups is None else (groups,)
    x = _randn((N, i), dtype, gen)
    w = _randn((*lead, o, i), dtype, gen, max(i, 1) ** -0.5)
    b = _randn((*lead, o), dtype, gen) if bias else None
    r = _randn((N, o), dtype, gen) if residual else None
    dy = _randn((N, o), dtype, gen)
    return x, w, b, r, dy


def _dev(t, grad=False):
    return None if t is None else t.to(DEV).requires_grad_(grad)


def _up(t):
    return None if t is None else t.double()


def _check(x, w, b, r, dy, act, edges=None, offsets=None, place=lambda t: t, on="cpu"):
    """Forward and backward of the operator against the definition, which is
    worked out ``on`` a device; ``place`` lays a device tensor out in memory."""
    from fedsim_amd.functional import grouped_linear, linear_act

    want = R.product(*(None if t is None else t.to(on).double() for t in (x, w, b, r)),
                     act, x.dtype, dy.to(on).double(), edges)
    leaves = [None if t is None else place(t.to(DEV)).requires_grad_(True) for t in (x, w, b, r)]
    X, W, B, Rr = leaves
    if edges is None:
        y = linear_act(X, W, B, Rr, activation=act)
    else:
        y = grouped_linear(X, W, offsets, B, Rr, activation=act)
    assert y.dtype == x.dtype and y.is_contiguous()
    R.close(y, want["y"], "y")
    have = [t for t in leaves if t is not None]
    grads = dict(zip([k for k, t in zip(("dx", "dw", "db", "dr"), leaves) if t is not None],
                     torch.autograd.grad(y, have, place(dy.to(DEV)))))
    for k in ("dx", "dw", "db"):
        if k in grads:
            assert grads[k].dtype == x.dtype
            R.close(grads[k], want[k], k)
    if "dr" in grads:
        assert torch.equal(grads["dr"].cpu(), dy)
    with torch.no_grad():  # the call that keeps nothing gives the same bits
        again = (linear_act(X, W, B, Rr, activation=act) if edges is None
                 else grouped_linear(X, W, offsets, B, Rr, activation=act))
    assert torch.equal(again.view(-1), y.detach().view(-1)) or again.isnan().any()
    return y, grads


SHAPES = [(1, 1, 1), (1, 784, 200), (2, 7, 9), (8, 513, 65), (9, 64, 1000), (16, 2048, 48),
          (33, 65, 129), (64, 128, 64), (100, 31, 300), (129, 256, 257), (257, 300, 70),
          (300, 520, 520), (1500, 72, 24), (3000, 8, 17), (40, 5000, 33)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear_shapes(shape, dtype):
    k = SHAPES.index(shape)
    act = ACTS[k % 4]
    x, w, b, r, dy = _case(*shape, dtype, k, bias=k % 3 != 1, residual=k % 2 == 0)
    _check(x, w, b, r, dy, act)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True),
                                           (True, True)])
def test_linear_epilogues(act, bias, residual, dtype):
    x, w, b, r, dy = _case(70, 96, 136, dtype, 5, bias=bias, residual=residual)
    _check(x, w, b, r, dy, act)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(0, 5, 7), (5, 0, 3), (3, 7, 0), (0, 0, 0)], ids=str)
def test_linear_empty(shape, dtype):
    for act in ACTS:
        _check(*_case(*shape, dtype, 1), act)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(640, 512, 768), (513, 1032, 520), (1024, 264, 1280)], ids=str)
def test_linear_large_tiles(shape, dtype):
    """Sizes that fill the widest tiles, with and without a remainder."""
    _check(*_case(*shape, dtype, 2), "gelu")
    _check(*_case(*shape, dtype, 3, bias=False, residual=False), "none")


@pytest.mark.parametrize("dtype,shape", [
    (torch.bfloat16, (4001, 3976, 4008)), (torch.float16, (4001, 3976, 4008)),
    (torch.bfloat16, (2600, 2051, 2049)), (torch.float16, (2600, 2051, 2049)),
    (torch.float32, (2600, 2051, 2049))], ids=str)
def test_linear_widest_tiles(dtype, shape):
    """Sizes at which each product takes the widest tiles there are for its type
    and alignment, with remainders."""
    _check(*_case(*shape, dtype, 4), "gelu", on=DEV)
    _check(*_case(*shape, dtype, 5, bias=False, residual=False), "none", on=DEV)


def _padded(t):
    """The same values in rows that lie further apart, one element off."""
    if t.dim() < 2:
        return torch.cat([t.new_zeros(1), t])[1:]
    wide = torch.full((*t.shape[:-1], t.shape[-1] + 3), float("nan"), dtype=t.dtype,
                      device=t.device)
    wide[..., 1:-2] = t
    return wide[..., 1:-2]


def _turned(t):
    """The same values, the last dimension not the closest."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t


def _wide(t):
    """Aligned rows with a gap of NaN behind each."""
    if t.dim() < 2:
        return t
    n = -(-t.shape[-1] // 8) * 8 + 16
    wide = torch.full((*t.shape[:-1], n), float("nan"), dtype=t.dtype, device=t.device)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("place", [_padded, _turned, _wide])
@pytest.mark.parametrize("shape", [(37, 200, 72), (3, 130, 264), (300, 256, 384)], ids=str)
def test_linear_strides(place, shape, dtype):
    _check(*_case(*shape, dtype, 6), "silu", place=place)
    x, w, b, r, dy = _case(*shape, dtype, 7, groups=3)
    off = [0, shape[0] // 3, shape[0] // 2, shape[0]]
    _check(x, w, b, r, dy, "gelu", off, torch.tensor(off, device=DEV), place=place)


def test_linear_leading_dimensions_and_broadcast():
    """x and residual of any leading dimensions; an expanded gradient and an
    expanded weight are read with their strides of 0."""
    from fedsim_amd.functional import grouped_linear, linear_act

    gen = torch.Generator().manual_seed(4)
    x, w, b, r, _ = _case(24, 40, 56, torch.float32, 8)
    for lead in ((), (24,), (4, 6), (2, 3, 4)):
        n = 24 if lead else 1
        X = x[:n].reshape(*lead, 40).to(DEV).requires_grad_(True)
        Rr = r[:n].reshape(*lead, 56).to(DEV)
        y = linear_act(X, w.to(DEV), b.to(DEV), Rr, activation="gelu")
        assert y.shape == (*lead, 56)
        want = R.product(_up(x[:n]), _up(w), _up(b), _up(r[:n]), "gelu", torch.float32,
                         torch.ones(n, 56, dtype=torch.float64))
        R.close(y.reshape(n, 56), want["y"], "y")
        y.sum().backward()  # the gradient of a sum is one value, expanded
        R.close(X.grad.reshape(n, 40), want["dx"], "dx")
    # one weight for every group, through expand: its gradient is the groups' sum
    W = _randn((56, 40), torch.float32, gen).to(DEV).requires_grad_(True)
    off = torch.tensor([0, 5, 24], device=DEV)
    y = grouped_linear(x.to(DEV), W.expand(2, 56, 40), off)
    want = R.product(_up(x), W.detach().double().cpu(), None, None, "none", torch.float32,
                     torch.ones(24, 56, dtype=torch.float64))
    R.close(y, want["y"], "y")
    y.sum().backward()
    v, e = want["dw"]
    R.close(W.grad, (v, 2 * e + 2.0 ** -23 * v.abs()), "dw")


GROUPS = [
    [3, 0, 5],
    [0, 0],
    [0],
    [7],
    [1] * 70,
    [200, 1, 63, 64, 65, 0, 129, 2],
    [16, 17, 15, 0, 0, 31, 32, 33, 128],
    [0, 0, 300, 0],
]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sizes", GROUPS, ids=lambda s: "-".join(map(str, s))[:24])
def test_grouped(sizes, dtype):
    k = GROUPS.index(sizes)
    for act, i, o, bias, residual in ((ACTS[k % 4], 72, 40, True, k % 2 == 0),
                                      (ACTS[(k + 1) % 4], 33, 131, False, k % 2 == 1)):
        edges = [0]
        for n in sizes:
            edges.append(edges[-1] + n)
        x, w, b, r, dy = _case(edges[-1], i, o, dtype, k, len(sizes), bias, residual)
        off = torch.tensor(edges, dtype=torch.int32 if k % 2 else torch.int64, device=DEV)
        _check(x, w, b, r, dy, act, edges, off)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("i,o", [(256, 320), (264, 136)])
def test_grouped_large_tiles(i, o, dtype):
    sizes = [300, 0, 513, 127, 1, 640]
    edges = [0]
    for n in sizes:
        edges.append(edges[-1] + n)
    x, w, b, r, dy = _case(edges[-1], i, o, dtype, 3, len(sizes))
    _check(x, w, b, r, dy, "silu", edges, torch.tensor(edges, device=DEV))


@pytest.mark.parametrize("dtype,i,o", [
    (torch.bfloat16, 1544, 1544), (torch.float16, 1544, 1544), (torch.bfloat16, 1535, 1281),
    (torch.float16, 1535, 1281), (torch.float32, 1535, 1281)], ids=str)
def test_grouped_widest_tiles(dtype, i, o):
    """As test_linear_widest_tiles, with a group of two thirds of the rows, an empty
    one, one of 70 and rows of no group."""
    edges = [1, 1500, 1500, 1570, 8191]
    N = 8192
    x, w, b, r, dy = _case(N, i, o, dtype, 12, 4)
    _check(x, w, b, r, dy, "silu", edges, torch.tensor(edges, device=DEV), on=DEV)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("groups", [1, 62, 63, 126, 127])
@pytest.mark.parametrize("i,o", [(40, 1104), (1101, 39)])
def test_grouped_many_tiles(groups, i, o, dtype):
    """More tiles than the card takes at a time, of as many ranges as are counted,
    or one more: groups of very different sizes, a third of them empty, rows
    before the first and behind the last."""
    gen = torch.Generator().manual_seed(groups)
    n = torch.exp(2 * torch.randn(groups, generator=gen)) * (torch.rand(groups, generator=gen) > .3)
    n[0] += 0.1
    edges = [3] + (3 + torch.round(n.cumsum(0) / n.sum() * 6990)).long().tolist()
    N = 7000
    x, w, b, r, dy = _case(N, i, o, dtype, 14, groups)
    _check(x, w, b, r, dy, "silu", edges, torch.tensor(edges, device=DEV), on=DEV)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("residual", [False, True])
def test_grouped_rows_of_no_group(dtype, residual):
    """Rows before the first and behind the last group: their residual or zero,
    no gradient for their x, and nothing of theirs in a weight's gradient (they
    hold NaN here)."""
    edges = [4, 30, 30, 101]
    x, w, b, r, dy = _case(140, 40, 72, dtype, 9, 3, True, residual)
    x[:4] = x[101:] = float("nan")
    clean = x.clone()
    clean[:4] = clean[101:] = 0
    want = R.product(_up(clean), _up(w), _up(b), _up(r), "gelu", dtype, _up(dy), edges)
    from fedsim_amd.functional import grouped_linear

    X, W, B = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    off = torch.tensor(edges, dtype=torch.int32, device=DEV)
    y = grouped_linear(X, W, off, B, _dev(r), activation="gelu")
    R.close(y, want["y"], "y")
    dx, dw, db = torch.autograd.grad(y, (X, W, B), dy.to(DEV))
    for g, k in ((dx, "dx"), (dw, "dw"), (db, "db")):
        R.close(g, want[k], k)
    outside = torch.cat([y[:4], y[101:]]).cpu()
    assert torch.equal(outside, torch.cat([r[:4], r[101:]]) if residual
                       else torch.zeros_like(outside))
    assert not torch.cat([dx[:4], dx[101:]]).any()


def test_grouped_offsets_outside_the_rows_are_cut():
    """Any values: the ranges are cut to the rows, an inverted one is empty."""
    from fedsim_amd.functional import grouped_linear

    x, w, b, _, dy = _case(50, 24, 40, torch.float32, 10, 3, True, False)
    for dt, edges, cut in ((torch.int64, [-7, 20, 1 << 40, 1 << 41], [0, 20, 50, 50]),
                           (torch.int32, [0, 10, 1000, 1 << 30], [0, 10, 50, 50])):
        W = w.to(DEV).requires_grad_(True)
        y = grouped_linear(x.to(DEV), W, torch.tensor(edges, dtype=dt, device=DEV), b.to(DEV))
        want = R.product(_up(x), _up(w), _up(b), None, "none", torch.float32, _up(dy), cut)
        R.close(y, want["y"], "y")
        R.close(torch.autograd.grad(y, W, dy.to(DEV))[0], want["dw"], "dw")


def test_grouped_weights_inside_a_slab():
    """A layer of K models whose flat vectors are the rows of one slab, where
    the layer starts at any element."""
    from fedsim_amd.functional import grouped_linear

    K, i, o, P = 5, 44, 30, 44 * 30 + 30 + 61
    gen = torch.Generator().manual_seed(1)
    for dtype in DTYPES:
        slab = _randn((K, P), dtype, gen, 0.1)
        dev = slab.to(DEV)
        for at in (0, 4, 33):
            w = slab[:, at:at + i * o].reshape(K, o, i)
            b = slab[:, at + i * o:at + i * o + o]
            x = _randn((64, i), dtype, gen)
            edges = [0, 9, 9, 40, 41, 64]
            y = grouped_linear(x.to(DEV), dev[:, at:at + i * o].unflatten(1, (o, i)),
                               torch.tensor(edges, device=DEV),
                               dev[:, at + i * o:at + i * o + o], activation="relu")
            R.close(y, R.product(_up(x), _up(w), _up(b), None, "relu", dtype, None, edges)["y"])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_infinities_and_nan_stay_where_they_belong(dtype):
    """A row of x with an infinity or NaN changes that row alone; a finite
    row's values near the type's largest do not overflow on the way."""
    x, w, b, _, dy = _case(70, 48, 33, dtype, 11, residual=False)
    w = w.abs() + 0.1
    x[3, 5], x[17, 0], x[40, 47] = float("inf"), float("-inf"), float("nan")
    big = torch.finfo(dtype).max
    x[50] = 0
    x[50, 7] = big
    w[:, 7] = 0.5
    for act in ("none", "relu"):
        want = R.product(_up(x), _up(w), _up(b), None, act, dtype)
        from fedsim_amd.functional import linear_act

        R.close(linear_act(x.to(DEV), w.to(DEV), b.to(DEV), activation=act), want["y"], act)
    # a gradient's NaN reaches its own row of dx, and its column of dW and db
    x, w, b, _, dy = _case(70, 48, 33, dtype, 12, residual=False)
    dy[9, 4] = float("nan")
    X, W, B = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    dx, dw, db = torch.autograd.grad(linear_act(X, W, B), (X, W, B), dy.to(DEV))
    assert dx.isnan().any(1).nonzero().view(-1).tolist() == [9]
    assert dw.isnan().any(1).nonzero().view(-1).tolist() == [4]
    assert db.isnan().nonzero().view(-1).tolist() == [4]


def test_subnormals_and_small_values():
    """float32 factors far below one keep float32's accuracy."""
    from fedsim_amd.functional import linear_act

    x, w, b, r, _ = _case(20, 64, 24, torch.float32, 13, bias=False, residual=False)
    for scale in (2.0 ** -60, 2.0 ** -20, 2.0 ** 40):
        X, W = x * scale, w * 2.0 ** -30
        y = linear_act(X.to(DEV), W.to(DEV))
        R.close(y, R.product(_up(X), _up(W), None, None, "none", torch.float32)["y"], str(scale))


def test_elements_past_32_bits():
    """Rows whose first element's number does not fit 31 bits."""
    from fedsim_amd.functional import linear_act

    N, i, o = 70_001, 32_768, 24
    x = torch.zeros(N, i, dtype=torch.float16, device=DEV)
    gen = torch.Generator().manual_seed(2)
    last = _randn((40, i), torch.float16, gen)
    w = _randn((o, i), torch.float16, gen, i ** -0.5)
    x[-40:] = last.to(DEV)
    W = w.to(DEV).requires_grad_(True)
    y = linear_act(x, W)
    R.close(y[-40:], R.product(_up(last), _up(w), None, None, "none", torch.float16)["y"], "y")
    assert not y[:-40].any()
    dy = torch.zeros_like(y)
    dy[-40:] = 1
    dw, = torch.autograd.grad(y, W, dy)
    want = R.product(_up(last), _up(w), None, None, "none", torch.float16,
                     torch.ones(40, o, dtype=torch.float64))["dw"]
    v, e = want
    R.close(dw, (v, e + R.sum_error(N, _up(last).abs().sum(0)[None].expand(o, i))), "dw")


def test_gradients_against_differences():
    """Central differences of a float32 forward pass: x is changed along one
    direction by +-d; the quotient is off by d^2 / 6 times the third derivative
    and by the forward's rounding over d."""
    from fedsim_amd.functional import grouped_linear

    x, w, b, r, dy = _case(40, 24, 16, torch.float32, 14, 2)
    off = torch.tensor([0, 13, 40], device=DEV)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b, r)]
    y = grouped_linear(leaves[0], leaves[1], off, leaves[2], leaves[3], activation="gelu")
    D = dy.to(DEV)
    grads = torch.autograd.grad(y, leaves, D)
    d = 2.0 ** -7
    gen = torch.Generator().manual_seed(3)
    for k, (leaf, g) in enumerate(zip(leaves, grads)):
        v = _randn(leaf.shape, torch.float32, gen).to(DEV)
        side = []
        for s in (d, -d):
            moved = [t.detach() + s * v if j == k else t.detach() for j, t in enumerate(leaves)]
            side.append((grouped_linear(moved[0], moved[1], off, moved[2], moved[3],
                                        activation="gelu").double() * D.double()).sum())
        slope = float((side[0] - side[1]) / (2 * d))
        want = float((g.double() * v.double()).sum())
        # 640 outputs of magnitude ~1, |dy| ~ 1, rounded to 2^-22 with random
        # signs: sqrt(640) 2^-22 / d < 1e-3; the third derivative (|gelu'''| < 1.2,
        # directions of size ~5 a row) gives sqrt(640) 125 d^2 / 6 < 0.04
        assert abs(slope - want) < 0.05, (k, slope, want)


def test_same_bits_every_time_and_on_another_stream():
    from fedsim_amd.functional import grouped_linear

    x, w, b, r, dy = _case(600, 136, 72, torch.bfloat16, 15, 7)
    off = torch.tensor([0, 100, 100, 300, 310, 311, 500, 600], device=DEV)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b, r)]
    D = dy.to(DEV)

    def once():
        y = grouped_linear(leaves[0], leaves[1], off, leaves[2], leaves[3], activation="gelu")
        return [y.detach(), *torch.autograd.grad(y, leaves, D)]

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, once()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    both = once()  # two calls under way at once
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(first, other))
    assert all(torch.equal(a, c) for a, c in zip(first, both))


def test_captured_and_replayed():
    """Forward and backward in one graph, replayed on new values and new
    offsets, with eager calls in between; a second graph beside it."""
    from fedsim_amd.functional import grouped_linear, linear_act

    def make(n, k):
        x, w, b, r, dy = _case(n, 96, 72, torch.float16, 16 + k, 4)
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b, r)]
        off = torch.tensor([0, n // 4, n // 4, n // 2, n], device=DEV)
        return leaves, off, dy.to(DEV)

    def once(leaves, off, dy):
        y = grouped_linear(leaves[0], leaves[1], off, leaves[2], leaves[3], activation="gelu")
        h = linear_act(y, leaves[1][0].t().contiguous(), activation="silu")
        return [h.detach(), *torch.autograd.grad(h, leaves[:3], dy[:, :1].expand(-1, 96))]

    graphs = []
    for k, n in enumerate((200, 1200)):
        leaves, off, dy = make(n, k)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            once(leaves, off, dy)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = once(leaves, off, dy)
        graphs.append((g, leaves, off, dy, out, n))
    for turn in range(3):
        for g, leaves, off, dy, out, n in graphs:
            with torch.no_grad():
                for t in leaves:
                    t.mul_(1.01)
            off.copy_(torch.tensor([0, turn, n // 3, n // 3 + turn, n - turn], device=DEV))
        for g, *_ in graphs:
            g.replay()
        for g, leaves, off, dy, out, n in graphs:
            now = once(leaves, off, dy)
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(out, now)), turn


def test_only_what_is_asked_for():
    """Any subset of the inputs may want a gradient."""
    from fedsim_amd.functional import linear_act

    x, w, b, r, dy = _case(50, 40, 24, torch.float32, 20)
    want = R.product(_up(x), _up(w), _up(b), _up(r), "silu", torch.float32, _up(dy))
    for mask in range(1, 16):
        t = [v.to(DEV).requires_grad_(bool(mask >> j & 1)) for j, v in enumerate((x, w, b, r))]
        y = linear_act(*t, activation="silu")
        asked = [v for v in t if v.requires_grad]
        grads = torch.autograd.grad(y, asked, dy.to(DEV))
        names = [n for j, n in enumerate(("dx", "dw", "db", "dr")) if mask >> j & 1]
        for n, g in zip(names, grads):
            if n == "dr":
                assert torch.equal(g.cpu(), dy)
            else:
                R.close(g, want[n], n)


def test_a_second_derivative_is_refused():
    from fedsim_amd.functional import linear_act

    x, w, b, _, dy = _case(20, 24, 16, torch.float32, 21, residual=False)
    X, W, B = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    y = linear_act(X, W, B, activation="gelu")
    dx, dw, db = torch.autograd.grad(y, (X, W, B), dy.to(DEV), create_graph=True)
    want = R.product(_up(x), _up(w), _up(b), None, "gelu", torch.float32, _up(dy))
    for g, k in ((dx, "dx"), (dw, "dw"), (db, "db")):
        R.close(g, want[k], k)
    with pytest.raises(RuntimeError, match="once"):
        (dx.sum() + dw.sum() + db.sum()).backward()


def test_gradients_accumulate_and_a_changed_input_is_noticed():
    from fedsim_amd.functional import linear_act

    x, w, b, _, dy = _case(20, 24, 16, torch.float32, 22, residual=False)
    X, W = (t.to(DEV).requires_grad_(True) for t in (x, w))
    for _ in range(2):
        linear_act(X, W, activation="silu").backward(dy.to(DEV))
    want = R.product(_up(x), _up(w), None, None, "silu", torch.float32, _up(dy))
    for g, k in ((X.grad, "dx"), (W.grad, "dw")):
        v, e = want[k]
        R.close(g, (2 * v, 2 * e + 2.0 ** -23 * v.abs()), k)
    y = linear_act(X, W)
    with torch.no_grad():
        W.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_negated_views_and_forward_mode():
    """A tensor whose sign torch has put off is read with it; a forward-mode
    derivative, which would be lost, raises."""
    import torch.autograd.forward_ad as fwad

    from fedsim_amd.functional import linear_act

    gen = torch.Generator().manual_seed(21)
    z = torch.randn(6, 5, generator=gen, dtype=torch.complex64).to(DEV)
    x, w = z.conj().imag, _dev(_randn((4, 5), torch.float32, gen))
    assert x.is_neg()
    assert torch.equal(linear_act(x, w), linear_act(x.resolve_neg().contiguous(), w))
    x = x.resolve_neg().contiguous()
    with fwad.dual_level():
        for a, b in ((fwad.make_dual(x, x), w), (x, fwad.make_dual(w, w))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                linear_act(a, b)


def test_two_at_once():
    """Calls with workspaces (k in parts) on two streams at the same time, eager and
    from two graphs: each has its own."""
    from fedsim_amd.train_ops import product_forward, product_grad_weight

    gen = torch.Generator().manual_seed(17)
    sets = [(_randn((40, 5000), torch.bfloat16, gen).to(DEV),
             _randn((96, 5000), torch.bfloat16, gen).to(DEV)) for _ in range(2)]

    def run(x, w):
        return [product_forward(x, w)[0],
                product_grad_weight(x.t().contiguous(), w.t().contiguous())[0]]

    want = [[t.cpu() for t in run(*s)] for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    graphs, kept = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kept.append(run(*s))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append([run(*s) for _ in range(4)][-1])
        torch.cuda.synchronize()
        for outs, w in zip(got, want):
            assert all(torch.equal(a.cpu(), b) for a, b in zip(outs, w))
        for outs in kept:
            for t in outs:
                t.zero_()
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for outs, w in zip(kept, want):
            assert all(torch.equal(a.cpu(), b) for a, b in zip(outs, w))
