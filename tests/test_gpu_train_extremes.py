"""linear_act and act_backward where a type's range or a formula's cancellation
decides: sums past float16, the far tails of the activations."""
import math

import pytest
import torch

import train_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda"


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act,below,above", [("none", 1, 1), ("relu", 0, 1), ("gelu", 0, 1),
                                             ("silu", 0, 1)])
def test_slopes_at_infinities(act, below, above, dtype):
    """A z that its type holds as an infinity has the slope of the far ends; a
    NaN has one of its own, or none."""
    from fedsim_amd.train_ops import act_backward

    inf = float("inf")
    z = torch.tensor([[-inf, inf, -inf, inf, -1.0, 1.0, torch.finfo(dtype).min,
                       torch.finfo(dtype).max]] * 3, dtype=dtype, device=DEV)
    dy = torch.full_like(z, 3.0)
    dz = act_backward(dy, z, act).cpu().double()
    for k in (0, 2, 6):
        assert (dz[:, k] == 3.0 * below).all(), (k, dz[0])
    for k in (1, 3, 7):
        assert (dz[:, k] == 3.0 * above).all(), (k, dz[0])


@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("residual", [False, True])
def test_float16_sums_past_its_range(act, residual):
    """Sums of +-70400 and more in float16: act(-70400) is 0 and act(70400)
    float16's infinity, with slopes of 0 and 1, so every gradient is finite and
    exact.  Everything is a sum of few small whole numbers."""
    from fedsim_amd.functional import linear_act

    x = torch.zeros(8, 16, dtype=torch.float16)
    x[:, 0] = torch.tensor([704., -704, 800, -800, 4, -1000, 1000, 0])
    x[:, 1] = 1
    w = torch.zeros(8, 16, dtype=torch.float16)
    w[:, 0] = 100  # every row's sums are 100 x0: +-70400, +-80000, 400, +-100000, 0
    dy = torch.ones(8, 8, dtype=torch.float16)
    dy[:, 3] = 2
    r = torch.full((8, 8), 5.0, dtype=torch.float16) if residual else None
    X, W = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    B = torch.zeros(8, dtype=torch.float16, device=DEV, requires_grad=True)
    y = linear_act(X, W, B, None if r is None else r.to(DEV), activation=act)
    z = 100.0 * x[:, :1].double().expand(8, 8)
    want = R.act(z, act) + (5.0 if residual else 0.0)
    assert torch.equal(y.detach().cpu(), want.to(torch.float16))
    dx, dw, db = torch.autograd.grad(y, (X, W, B), dy.to(DEV))
    slope = R.slope(z, act)
    dz = dy.double() * slope
    assert torch.equal(dx.cpu().double(), (dz @ w.double()))
    assert torch.equal(dw.cpu().double(), (dz.T @ x.double()))
    assert torch.equal(db.cpu().double(), dz.sum(0))


def _tail_error(z):
    """How far Phi(z) and z phi(z) in float32 may be off, relative: 13 units of
    2^-24 for the approximation, 24 for its terms' roundings and the hardware's
    reciprocal and exponential, and z^2 / 2, the exponent, off by 4.5 units of its
    own; a library's erfc takes 32 and an argument rounded once."""
    return (40 + 4 * z * z) * 2.0 ** -24


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gelus_tail(dtype):
    """gelu(z) = z Phi(z) and its slope are good relative to themselves for
    negative z too, where 1 + erf(z / sqrt 2) cancels."""
    from fedsim_amd.functional import linear_act
    from fedsim_amd.train_ops import act_backward

    low = {torch.float32: -12.5, torch.bfloat16: -12.5, torch.float16: -6.0}[dtype]
    z = torch.linspace(low, 6.0, 20_011, dtype=torch.float64).to(dtype)
    y = linear_act(z[:, None].to(DEV), torch.ones(1, 1, dtype=dtype, device=DEV),
                   activation="gelu")
    z = z.double()
    cdf = torch.erfc(z * -math.sqrt(0.5)) / 2  # torch's ndtr cancels below -8
    far = z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    want = z * cdf
    e = _tail_error(z) * want.abs()
    R.close(y[:, 0], (want, e + R.HALF[dtype] * (want.abs() + e) + R.TINY[dtype]), "gelu")
    dz = act_backward(torch.ones(1, z.numel(), dtype=dtype, device=DEV),
                      z.to(dtype)[None].to(DEV), "gelu")
    want = cdf + far
    e = _tail_error(z) * (cdf + far.abs())
    R.close(dz[0], (want, e + R.HALF[dtype] * (want.abs() + e) + R.TINY[dtype]), "slope")


def test_float32_products_of_few_terms():
    """float32 products in three bf16 parts, for sums too short to hide what is
    left out: 2^-24 of each product, (1 + 2^-9) of it.  A sum of K takes 2^-23
    for each addition where the matrix unit cuts off, and the smaller parts' own
    sums, at most 2^-6 of it in four instructions, 2^-27."""
    from fedsim_amd.functional import linear_act
    from fedsim_amd.train_ops import product_grad_weight

    gen = torch.Generator().manual_seed(31)
    for K in (1, 2, 3):
        x = torch.randn(K, 700, generator=gen)
        d = torch.randn(K, 300, generator=gen)
        dw, _ = product_grad_weight(d.to(DEV), x.to(DEV))
        S = d.double().abs().T @ x.double().abs()
        e = (2.0 ** -24 + 2.0 ** -23 * K + 2.0 ** -26) * S
        R.close(dw, (d.double().T @ x.double(), e), f"dw {K}")
        a, b = x.T.contiguous(), d.T.contiguous()
        y = linear_act(a.to(DEV), b.to(DEV))
        R.close(y, (a.double() @ b.double().T, e.T), f"y {K}")


@pytest.mark.parametrize("tiny", [2.0 ** -100, 2.0 ** -112, 2.0 ** -120, 2.0 ** -126, 2.0 ** -135])
def test_float32_factors_next_to_the_smallest(tiny):
    """A factor's bf16 parts below 2^-126 may be lost: two of them at most, the
    larger below 2^-126 and the other 2^-8 of it, so a factor is off by 2^-125
    at most, next to the rounding of normal sums."""
    from fedsim_amd.functional import linear_act

    gen = torch.Generator().manual_seed(32)
    x = torch.randn(40, 64, generator=gen).double() * tiny
    x = x.to(torch.float32)  # subnormals for the last two
    w = torch.randn(24, 64, generator=gen)
    y = linear_act(x.to(DEV), w.to(DEV))
    S = x.double().abs() @ w.double().abs().T
    e = R.sum_error(64, S) + 2.0 ** -125 * w.double().abs().sum(1)[None] + 64 * R.TINY[torch.float32]
    R.close(y, (x.double() @ w.double().T, e.expand(40, 24)), str(tiny))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_the_call_that_keeps_nothing_gives_the_same_bits(act, dtype):
    """With autograd off no z is stored; NaN are where they were."""
    from fedsim_amd.functional import linear_act

    gen = torch.Generator().manual_seed(33)
    for N, K, M in ((3, 40, 70), (70, 96, 136), (600, 520, 520), (300, 33, 129)):
        x = torch.randn(N, K, generator=gen).to(dtype)
        x[N // 2, 1], x[0, 3] = float("nan"), float("inf")
        w = torch.randn(M, K, generator=gen).to(dtype).to(DEV)
        b = torch.randn(M, generator=gen).to(dtype).to(DEV)
        r = torch.randn(N, M, generator=gen).to(dtype).to(DEV)
        X = x.to(DEV).requires_grad_(True)
        kept = linear_act(X, w, b, r, activation=act).detach()
        with torch.no_grad():
            bare = linear_act(X, w, b, r, activation=act)
        assert kept[N // 2].isnan().all()
        i = torch.int32 if dtype == torch.float32 else torch.int16
        assert torch.equal(kept.isnan(), bare.isnan())
        assert torch.equal(kept.nan_to_num(7.0).view(i), bare.nan_to_num(7.0).view(i))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("case", [(777, 333, None), (1, 40, None), (2048, 65, None),
                                  (2049, 8, None), (9000, 130, None), (0, 9, None),
                                  (700, 136, [0, 300, 300, 301, 700]),
                                  (9000, 70, [5, 2100, 2100, 8800]), (64, 12, [0] * 40 + [60])],
                         ids=str)
def test_bias_gradients_are_sums_of_unrounded_terms(case, act, dtype):
    """db in 16 bits: the terms dy act'(z) are not rounded on their way.  x is one
    value a row and w is 1, so z is x, which its type holds: float32's slope (16
    units of 2^-24 of 1 + |z|, and relu's none) and sum are all that is between db
    and the definition's, rounded once."""
    from fedsim_amd.functional import grouped_linear, linear_act

    N, M, edges = case
    gen = torch.Generator().manual_seed(N + M)
    x = torch.randn(N, 1, generator=gen).to(dtype)
    dy = torch.randn(N, M, generator=gen).to(dtype)
    G = len(edges) - 1 if edges else 1
    w = torch.ones(G, M, 1, dtype=dtype, device=DEV)
    B = torch.zeros(G, M, dtype=dtype, device=DEV, requires_grad=True)
    X = x.to(DEV).requires_grad_(True)
    if edges:
        y = grouped_linear(X, w, torch.tensor(edges, device=DEV), B, activation=act)
    else:
        y = linear_act(X, w[0], B[0], activation=act)
    db, dx = torch.autograd.grad(y, (B, X), dy.to(DEV))
    z = x.double().expand(N, M)
    dz = dy.double() * R.slope(z, act)
    unit = 0.0 if act == "relu" else 16 * 2.0 ** -24
    term = dy.double().abs() * unit * (1 + z.abs())
    for g, (lo, hi) in enumerate(zip(edges, edges[1:]) if edges else [(0, N)]):
        v, s = dz[lo:hi].sum(0), dz[lo:hi].abs().sum(0)
        e = term[lo:hi].sum(0) + R.sum_error(hi - lo, s)
        R.close(db[g], (v, e + R.HALF[dtype] * (v.abs() + e) + R.TINY[dtype]), f"db {g}")
        if hi == lo:
            assert not db[g].any()
    again = torch.autograd.grad(
        grouped_linear(X, w, torch.tensor(edges, device=DEV), B, activation=act) if edges
        else linear_act(X, w[0], B[0], activation=act), B, dy.to(DEV))[0]
    assert torch.equal(again, db)
