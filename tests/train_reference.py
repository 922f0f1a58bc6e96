"""The dense training operators from their definitions, in 64 bits, with bounds on how far a float32-summed kernel may be from them.

Bounds.  A value stored in a type t is off by at most h = eps(t) / 2 relative to
it.  A sum of K products in float32, in any order, is off by at most
(K + 2) 2^-23 S with S the sum of the magnitudes (2^-24 an operation in round to
nearest; 2^-23 allows the matrix units to cut off instead, and covers an exact
split of float32 factors into three 8-bit parts whose smallest products, below
2^-21 S, are left out).  Activations have slopes within 1.13 and second
derivatives within 0.8 (gelu) and 0.5 (silu); evaluating one in float32 costs at
most 16 units of 2^-24 of its argument's magnitude.
"""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half the spacing of the subnormals: what a value near zero is off by
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def act(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.where(z.isnan(), z, 0.0))
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    if kind == "silu":
        return z * torch.special.expit(z)
    return z


def slope(z, kind):
    if kind == "relu":
        return (z > 0).double()
    if kind == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "silu":
        s = torch.special.expit(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


CURVE = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "silu": 0.5}


def sum_error(K, S):
    return (K + 8) * 2.0 ** -23 * S


def product(x, w, b, r, kind, dtype, dy=None, edges=None):
    """{name: (value, bound)} of y, dx, dw, db for float64 tensors of one device;
    ``edges``: the groups' row bounds (w and b then have a group dimension)."""
    h, t = HALF[dtype], TINY[dtype]
    N, o = x.shape[0], w.shape[-2]
    grouped = edges is not None
    if not grouped:
        edges, w, b = [0, N], w[None], None if b is None else b[None]
    G = len(edges) - 1
    y = torch.zeros(N, o, dtype=torch.float64, device=x.device) if r is None else r.clone()
    ey = h * y.abs()
    out = {}
    if dy is not None:
        dx, edx = torch.zeros_like(x), torch.zeros_like(x)
        dw, edw = torch.zeros_like(w), torch.zeros_like(w)
        db = torch.zeros(G, o, dtype=torch.float64, device=x.device)
        edb = torch.zeros_like(db)
    for g in range(G):
        s = slice(edges[g], max(edges[g], edges[g + 1]))
        X, W = x[s], w[g]
        K = X.shape[1]
        z = X @ W.T
        S = X.abs() @ W.abs().T
        if b is not None:
            z, S = z + b[g], S + b[g].abs()
        ez = sum_error(K, S) + t
        v = act(z, kind)
        e = 1.13 * ez + 16 * 2.0 ** -24 * z.abs()
        if r is not None:
            v = v + r[s]
            e = e + 2.0 ** -23 * (v.abs() + r[s].abs())
        y[s] = v
        ey[s] = e + h * (v.abs() + e) + t
        if dy is None:
            continue
        D = dy[s]
        if kind == "none":
            dz, edz = D, torch.zeros_like(D)
        else:
            sl = slope(z, kind)
            dz = D * sl
            es = CURVE[kind] * (ez + h * (z.abs() + ez) + t) + 16 * 2.0 ** -24 * (1 + z.abs())
            if kind == "relu":  # within the sum's error of 0 either side is right
                es = torch.where(z.abs() <= ez, 1.0, 0.0)
            edz = D.abs() * es
            edz = edz + h * (dz.abs() + edz) + t
        top = dz.abs() + edz
        v = dz @ W
        e = edz @ W.abs() + sum_error(o, top @ W.abs())
        dx[s], edx[s] = v, e + h * (v.abs() + e) + t
        n = X.shape[0]
        v = dz.T @ X
        e = edz.T @ X.abs() + sum_error(n, top.T @ X.abs())
        dw[g], edw[g] = v, e + h * (v.abs() + e) + t
        v = dz.sum(0)
        e = edz.sum(0) + sum_error(n, top.sum(0))
        db[g], edb[g] = v, e + h * (v.abs() + e) + t
    out["y"] = (y, ey)
    if dy is not None:
        if not grouped:
            dw, edw, db, edb = dw[0], edw[0], db[0], edb[0]
        out.update(dx=(dx, edx), dw=(dw, edw), db=(db, edb))
    return out


def close(got, want, what=""):
    value, bound = want
    got = got.detach().double().to(value.device)
    assert got.shape == value.shape, (what, got.shape, value.shape)
    if not got.numel():
        return
    finite = value.isfinite()
    assert bool((got.isfinite() == finite).all()), f"{what}: infinities or NaN differ"
    assert bool((got.isnan() == value.isnan()).all()), f"{what}: NaN differ"
    inf = ~finite & ~value.isnan()
    assert bool((got[inf] == value[inf]).all()), f"{what}: signs of infinities differ"
    off = torch.where(finite, (got - value).abs() - bound, -1.0)
    worst = int(off.argmax())
    assert float(off.max()) <= 0, (
        f"{what}: {got.reshape(-1)[worst]} for {value.reshape(-1)[worst]}, "
        f"allowed {bound.reshape(-1)[worst]}; {int((off > 0).sum())} of {off.numel()} are off")


# ---------------------------------------------------------------------------
# the AdamW step
# ---------------------------------------------------------------------------
BLOCK = 256


def mix(h):
    h = h ^ (h >> 16)
    h = (h * 0x6A09E667) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0xBB67AE85) & 0xFFFFFFFF
    return h ^ (h >> 16)


def moments32(m, v, g, betas):
    """The new moments with float32's rounding of each product and sum."""
    b1, c1, b2, c2 = (torch.tensor(x, dtype=torch.float32)
                      for x in (betas[0], 1 - betas[0], betas[1], 1 - betas[1]))
    return m * b1 + g * c1, v * b2 + (g * c2) * g


def blocks_of(x):
    n = x.numel()
    pad = -n % BLOCK
    return torch.cat([x.reshape(-1), x.new_zeros(pad)]).view(-1, BLOCK)


def _power(biased):
    return torch.bitwise_left_shift(biased.to(torch.int32), 23).view(torch.float32)


def _biased(x):
    return torch.bitwise_right_shift(x.contiguous().view(torch.int32), 23)


def quantize(x, top, mantissa, least, u, floor=False):
    """(codes as float32 values, scales) of a float32 tensor's blocks."""
    x = blocks_of(x)
    finite = torch.where(x.isfinite(), x.abs(), 0.0)
    scale = _power((_biased(finite.amax(1) * 0.57735026918962576) - top).clamp(min=1))
    a = torch.where(x.isfinite(), x.abs(), 0.0) / scale[:, None]
    e = _biased(a).clamp(min=127 + least)
    step = _power(e - mantissa)
    q = torch.floor(a / step + u.float() * 2.0 ** -16) * step
    if floor:
        q = torch.where(a > 0, q.clamp(min=2.0 ** -16), q)
    return torch.copysign(q, x), scale


def states8(m, v, step, seed, block0=0):
    """(m codes, m scales, v codes, v scales) of the new moments of one tensor."""
    nb = -(-m.numel() // BLOCK)
    key = int(mix(torch.tensor((seed & 0xFFFFFFFF)) ^ mix(torch.tensor(step & 0xFFFFFFFF))))
    bk = mix((key + (torch.arange(nb) + block0) * 0x9E3779B9) & 0xFFFFFFFF)
    h = mix((bk[:, None] + torch.arange(BLOCK) * 0x9E3779B9) & 0xFFFFFFFF)
    qm, sm = quantize(m, 7, 3, -6, h & 0xFFFF)
    qv, sv = quantize(v, 14, 2, -14, h >> 16, floor=True)
    n = m.numel()
    return qm.view(-1)[:n], sm, qv.view(-1)[:n], sv
