"""The dense training operators as they are measured: a matrix product with its
epilogue, matrix products grouped by client, and the AdamW step.

``listed()`` and ``draw()`` give cases, ``prepare()`` a case's inputs on the GPU,
``run()`` one pass: in plain torch operations, or with ``own`` set through
``fedsim_amd``.  ``exact()`` is the same from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01
BLOCK = 256  # elements that share a scale where states are held in 8 bits
MLP = (156800, 200, 40000, 200, 2000, 10)  # SimpleMLP: fc1, fc2, classifier


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _linear(rows, inp, out, dtype, act, bias, residual, train):
    return dict(kind="linear", rows=rows, inp=inp, out=out, dtype=dtype, act=act, bias=bias,
                residual=residual, train=train)


def _grouped(groups, rows, inp, out, dtype, act, bias, residual, train, spread, tail=0):
    """``rows`` in all; group sizes are lognormal with sigma ``spread``, some
    groups of a wide spread are empty; ``tail`` rows belong to no group: they
    get no product, and their residual or zero."""
    return dict(kind="grouped", groups=groups, rows=rows, inp=inp, out=out, dtype=dtype, act=act,
                bias=bias, residual=residual, train=train, spread=spread, tail=tail)


def _adamw(tensors, elements, dtype, state_bits):
    return dict(kind="adamw", tensors=tensors, elements=elements, dtype=dtype,
                state_bits=state_bits)


def listed():
    return [
        # SimpleMLP's first layer, one client's batch: launches and latency
        dict(_linear(32, 784, 200, "f32", "relu", True, False, True), name="linear 2NN batch"),
        # one token through a square layer: the weights are read once
        dict(_linear(1, 4096, 4096, "bf16", "silu", True, True, False), name="linear one row"),
        # nothing is a multiple of anything
        dict(_linear(777, 1001, 333, "f16", "gelu", True, True, True), name="linear odd"),
        # SimpleCNN's wide layer (3136 -> 512) over a large server batch, in the simulator's type
        dict(_linear(2048, 3136, 512, "f32", "silu", True, False, True), name="linear f32"),
        # a feed-forward layer of a large model, one training step
        dict(_linear(8192, 4096, 16384, "bf16", "gelu", True, False, True), name="linear large"),
        # ten clients' first layers, one ragged batch each
        dict(_grouped(10, 320, 784, 200, "f32", "relu", True, False, True, 0.5),
             name="grouped 2NN cohort"),
        # SimpleCNN2's fc1 of 1000 clients, each on its own samples: weights read once
        dict(_grouped(1000, 48000, 2304, 384, "f32", "relu", True, False, False, 0.5),
             name="grouped 1000 clients"),
        # experts of a large layer, one training step
        dict(_grouped(64, 16384, 2048, 5632, "bf16", "silu", False, False, True, 0.5),
             name="grouped experts"),
        # odd sizes, empty groups, rows behind the last group
        dict(_grouped(37, 3001, 1003, 517, "f16", "gelu", True, True, True, 1.0, 17),
             name="grouped odd"),
        # SimpleMLP's six tensors: launches and latency
        dict(_adamw(6, sum(MLP), "f32", 32), name="adamw 2NN"),
        # a 25 M parameter model held in bf16, states in 8 bits
        dict(_adamw(60, 25_000_000, "bf16", 8), name="adamw 25M 8 bit"),
        # a 125 M parameter vector, states in 32 bits
        dict(_adamw(1, 125_000_000, "f32", 32), name="adamw 125M"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Spread over the logarithm; half of them multiples of 64, half anything."""
    n = _log(rng, lo, hi)
    return max(lo, n // 64 * 64) if rng.random() < 0.5 and n >= 64 else n


def draw(rng):
    kind = rng.choice(("linear", "grouped", "adamw"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if kind == "adamw":
        return _adamw(rng.randint(1, 80), _log(rng, 20_000, 100_000_000), dtype,
                      rng.choice((8, 32)))
    act = rng.choice(("none", "relu", "gelu", "silu"))
    bias, residual, train = (rng.random() < 0.5 for _ in range(3))
    if kind == "linear":
        rows, inp, out = _log(rng, 1, 8192), _size(rng, 16, 8192), _size(rng, 10, 8192)
        if act == "relu" and dtype == "f32" and train and rows * out > 50_000:
            act = "silu"  # a gradient that jumps at 0 says nothing near 0
        return _linear(rows, inp, out, dtype, act, bias, residual, train)
    groups, inp, out = _log(rng, 2, 512), _size(rng, 16, 4096), _size(rng, 10, 4096)
    while groups * inp * out > 600_000_000:
        groups = max(1, groups // 2)
    rows = min(16384, groups * _log(rng, 1, 512))
    if act == "relu" and dtype == "f32" and train and rows * out > 50_000:
        act = "silu"
    return _grouped(groups, rows, inp, out, dtype, act, bias, residual, train,
                    rng.choice((0.2, 0.5, 1.0)), rng.choice((0, 0, 5)))


def _sizes(case):
    """Lengths of the optimizer's tensors: a model's mix of large weights and
    short vectors, the same for every seed."""
    n, total = case["tensors"], case["elements"]
    if (n, total) == (len(MLP), sum(MLP)):
        return list(MLP)
    w = np.random.RandomState(n).lognormal(0.0, 1.5, n)
    w[1::2] *= 1e-3  # biases
    s = np.maximum(1, np.floor(w / w.sum() * total)).astype(np.int64)
    s[0] += max(0, total - int(s.sum()))
    return [int(v) for v in s]


def _group_sizes(case, seed):
    r = np.random.RandomState(seed % (1 << 31))
    w = r.lognormal(0.0, case["spread"], case["groups"])
    if case["spread"] >= 1.0:
        w[r.rand(case["groups"]) < 0.1] = 0.0
        w[0] = max(w[0], 0.1)
    edges = np.round(np.cumsum(w) / w.sum() * case["rows"]).astype(np.int64)
    return np.diff(np.concatenate([[0], edges]))


def work(case):
    if case["kind"] == "adamw":
        n, b = sum(_sizes(case)), BYTES[case["dtype"]]
        state = 8 if case["state_bits"] == 32 else 2 + 8 / BLOCK
        return {"bytes": n * (3 * b + 2 * state), "flops": 16.0 * n}
    n, i, o, b = case["rows"], case["inp"], case["out"], BYTES[case["dtype"]]
    g = case.get("groups", 1)
    total = n + case.get("tail", 0)
    w, x, y = g * o * i, total * i, total * o
    vec = g * o if case["bias"] else 0
    res = y if case["residual"] else 0
    size, flops = w + x + y + vec + res, 2.0 * n * i * o
    if case["train"]:  # dy and the saved z (or y) in, dx, dW, db out
        size += (y + w + x) + (y if case["act"] != "none" else 0) + (x + w + vec)
        flops *= 3
    return {"bytes": size * b, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dt)

    s = dict(case=case)
    if case["kind"] == "adamw":
        return _prepare_adamw(s, case, gen, dt)
    i, o, total = case["inp"], case["out"], case["rows"] + case.get("tail", 0)
    lead = ()
    if case["kind"] == "grouped":
        lead = (case["groups"],)
        sizes = _group_sizes(case, seed)
        s["most"] = int(sizes.max())  # rows of the largest group: the program dealt them out
        s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)])).to("cuda",
                                                                                   torch.int32)
    s["x"] = randn(total, i)
    s["w"] = randn(*lead, o, i, scale=1 / math.sqrt(i))
    s["b"] = randn(*lead, o, scale=0.1) if case["bias"] else None
    s["r"] = randn(total, o) if case["residual"] else None
    if case["train"]:
        s["dy"] = randn(total, o)
        for k in ("x", "w", "b", "r"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def _exponent(t):
    """Biased exponents of non-negative f32 values."""
    return torch.bitwise_right_shift(t.view(torch.int32), 23)


def _power(biased):
    return torch.bitwise_left_shift(biased, 23).view(torch.float32)


def _scale(most, top):
    """A block's power of two, from its largest magnitude: that magnitude over
    it lies between sqrt(3) 2^top and sqrt(3) 2^(top + 1): a border that sums of
    codes and decimals do not meet."""
    return _power((_exponent(most * (1 / math.sqrt(3))) - top).clamp(min=1))


def _views(flat, case):
    views, at = [], 0
    for n in _sizes(case):
        views.append(flat[at:at + n])
        at += -(-n // BLOCK) * BLOCK
    return views


def _scale_views(flat, case):
    views, at = [], 0
    for n in _sizes(case):
        views.append(flat[at:at + -(-n // BLOCK)])
        at += -(-n // BLOCK)
    return views


def _prepare_adamw(s, case, gen, dt):
    """Parameters, gradients and states in the middle of a training run.  The
    tensors lie one after another, each begun at a multiple of 256 elements."""
    blocks = sum(-(-n // BLOCK) for n in _sizes(case))
    n = blocks * BLOCK
    inside = torch.zeros(n, device="cuda")
    for v in _views(inside, case):
        v.fill_(1.0)
    size = torch.exp(torch.randn(n, generator=gen, device="cuda")) * 1e-3 * inside
    s["p"] = (torch.randn(n, generator=gen, device="cuda") * 0.05 * inside).to(dt)
    s["g"] = (torch.randn(n, generator=gen, device="cuda") * size).to(dt)
    m = torch.randn(n, generator=gen, device="cuda") * size * 0.3
    v = size * size * (0.5 + torch.rand(n, generator=gen, device="cuda"))
    if case["state_bits"] == 8:
        ms = _scale(m.abs().view(-1, BLOCK).amax(1), 7)
        vs = _scale(v.view(-1, BLOCK).amax(1), 14)
        m = (m.view(-1, BLOCK) / ms[:, None]).view(-1).to(torch.float8_e4m3fn)
        v = (v.view(-1, BLOCK) / vs[:, None]).view(-1).to(torch.float8_e5m2)
        s["ms"], s["vs"] = ms, vs
        s["ms_list"], s["vs_list"] = _scale_views(ms, case), _scale_views(vs, case)
    s["m"], s["v"] = m, v
    for k in ("p", "g", "m", "v"):
        s[k + "_list"] = _views(s[k], case)
    s["step"] = 100
    s["seed"] = 1234
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if s["case"]["kind"] == "adamw":
        s["step"] += 1
        if own:
            _own_adamw(s)
        else:
            _plain_adamw(s)
        return {k: s[k] for k in ("p", "m", "v", "ms", "vs") if k in s}
    if own:
        return _own_product(s)
    with torch.no_grad():
        return _plain_product(s)


def _own_product(s):
    from fedsim_amd.functional import grouped_linear, linear_act

    case = s["case"]
    if case["kind"] == "grouped":
        y = grouped_linear(s["x"], s["w"], s["offsets"], s["b"], s["r"], activation=case["act"])
    else:
        y = linear_act(s["x"], s["w"], s["b"], s["r"], activation=case["act"])
    out = {"y": y.detach()}
    if case["train"]:
        names = [k for k in ("x", "w", "b", "r") if s[k] is not None]
        for k, g in zip(names, torch.autograd.grad(y, [s[k] for k in names], s["dy"])):
            out["d" + k] = g
    return out


def _own_adamw(s):
    from fedsim_amd.train_ops import adamw_step

    adamw_step(s["p_list"], s["g_list"], s["m_list"], s["v_list"], s.get("ms_list"),
               s.get("vs_list"), step=s["step"], lr=LR, betas=BETAS, eps=EPS,
               weight_decay=DECAY, seed=s["seed"])


def _act(z, kind):
    if kind == "relu":
        return z.clamp(min=0)
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + \
            z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if kind == "silu":
        t = 1 / (1 + torch.exp(-z))
        return t * (1 + z * (1 - t))
    return torch.ones_like(z)


def _plain_product(s):
    """In 32 bits, rounded at the end; grouped rows go through products padded
    to the largest group."""
    case = s["case"]
    dt, kind, train = DTYPES[case["dtype"]], case["act"], case["train"]
    x, w = s["x"].float(), s["w"].float()
    grouped = case["kind"] == "grouped"
    if grouped:
        off = s["offsets"].long()
        N, G = x.shape[0], case["groups"]
        at = off[:-1, None] + torch.arange(s["most"], device=x.device)
        held = (at < off[1:, None]).unsqueeze(2)
        at = at.clamp(max=N - 1)
        row = torch.arange(N, device=x.device)
        of = torch.searchsorted(off[1:].contiguous(), row, right=True)
        inside = (of < G).unsqueeze(1)
        of = of.clamp(max=G - 1)
        place = (row - off[of]).clamp(min=0, max=max(0, s["most"] - 1))

        def deal(t):  # rows -> [G, most, ...], zeros behind a group's rows
            return torch.where(held, t[at], 0.0)

        def back(t):
            return torch.where(inside, t[of, place], 0.0)

        x = deal(x)
    z = x @ w.transpose(-1, -2)
    if s["b"] is not None:
        z = z + (s["b"].float().unsqueeze(1) if grouped else s["b"].float())
    y = _act(z, kind)
    if grouped:
        y = back(y)
    if s["r"] is not None:
        y = y + s["r"].float()
    out = {"y": y.to(dt)}
    if not train:
        return out
    dy = s["dy"].float()
    dz = deal(dy) if grouped else dy
    if kind != "none":
        dz = dz * _act_slope(z, kind)
    dx = dz @ w
    out["dx"] = (back(dx) if grouped else dx).to(dt)
    out["dw"] = (dz.transpose(-1, -2) @ x).to(dt)
    if s["b"] is not None:
        out["db"] = dz.sum(-2).to(dt)
    if s["r"] is not None:
        out["dr"] = s["dy"]
    return out


def _mix(h):
    """A 32-bit hash in 64-bit integers: two rounds of xor-shift and multiply."""
    h = h ^ (h >> 16)
    h = (h * 0x6A09E667) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0xBB67AE85) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _stochastic(x, scale, u, mantissa, least):
    """|x| / scale rounded to a float of ``mantissa`` bits and smallest normal
    2^least: up where the part cut off and u (16 bits over 2^16) reach one."""
    a = x.abs() / scale
    e = _exponent(a).clamp(min=127 + least)
    step = _power(e - mantissa)
    return torch.floor(a / step + u) * step


def _plain_adamw(s):
    b1, b2 = BETAS
    t = s["step"]
    p, g = s["p"].float(), s["g"].float()
    m, v = s["m"], s["v"]
    eight = "ms" in s
    if eight:
        m = (m.float().view(-1, BLOCK) * s["ms"][:, None]).view(-1)
        v = (v.float().view(-1, BLOCK) * s["vs"][:, None]).view(-1)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    root = v.sqrt() * (1 / math.sqrt(1 - b2 ** t)) + EPS
    p = p * (1 - LR * DECAY) - (m / root) * (LR / (1 - b1 ** t))
    s["p"].copy_(p)
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return
    blocks = s["ms"].numel()
    key = _mix(torch.tensor(s["seed"] & 0xFFFFFFFF) ^ _mix(torch.tensor(t & 0xFFFFFFFF)))
    key = _mix((int(key) + torch.arange(blocks, device=p.device) * 0x9E3779B9) & 0xFFFFFFFF)
    lane = torch.arange(BLOCK, device=p.device) * 0x9E3779B9
    h = _mix((key[:, None] + lane) & 0xFFFFFFFF)
    m, v = m.view(-1, BLOCK), v.view(-1, BLOCK)
    s["ms"].copy_(_scale(m.abs().amax(1), 7))
    s["vs"].copy_(_scale(v.amax(1), 14))
    qm = _stochastic(m, s["ms"][:, None], (h & 0xFFFF).float() * 2.0 ** -16, 3, -6)
    qv = _stochastic(v, s["vs"][:, None], (h >> 16).float() * 2.0 ** -16, 2, -14)
    qv = torch.where(v > 0, qv.clamp(min=2.0 ** -16), qv)
    s["m"].copy_(torch.copysign(qm, m).view(-1))
    s["v"].copy_(qv.view(-1))


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_adamw(s) if case["kind"] == "adamw" else _exact_product(s)


def _exact_product(s):
    case = s["case"]
    x, w = s["x"].double(), s["w"].double()
    N, o = x.shape[0], case["out"]
    G = case.get("groups", 1)
    edges = s["offsets"].tolist() if G > 1 or "offsets" in s else [0, N]
    w = w.view(G, o, -1)
    b = s["b"].double().view(G, o) if s["b"] is not None else None
    y = torch.zeros(N, o, dtype=torch.float64, device=x.device)
    if s["r"] is not None:
        y += s["r"].double()
    out = {"y": y}
    if case["train"]:
        dy = s["dy"].double()
        out["dx"], dw = torch.zeros_like(x), torch.zeros_like(w)
        db = torch.zeros(G, o, dtype=torch.float64, device=x.device)
    for k in range(G):
        rows = slice(edges[k], edges[k + 1])
        if edges[k + 1] == edges[k]:
            continue
        z = torch.mm(x[rows], w[k].t().contiguous())
        if b is not None:
            z += b[k]
        cdf = torch.special.ndtr(z)
        sig = torch.special.expit(z)
        value, slope = {
            "none": (z, None),
            "relu": (torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0)),
            "gelu": (z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)),
            "silu": (z * sig, sig + z * sig * (1 - sig)),
        }[case["act"]]
        y[rows] += value
        if case["train"]:
            dz = dy[rows] if slope is None else dy[rows] * slope.double()
            out["dx"][rows] = torch.mm(dz, w[k])
            dw[k] = torch.mm(dz.t().contiguous(), x[rows])
            db[k] = dz.sum(0)
    if case["train"]:
        out["dw"] = dw.view(s["w"].shape)
        if b is not None:
            out["db"] = db.view(s["b"].shape)
        if s["r"] is not None:
            out["dr"] = dy
    return out


def _hash32(h):
    h = h.astype(np.uint32)
    h ^= h >> np.uint32(16)
    h *= np.uint32(0x6A09E667)
    h ^= h >> np.uint32(15)
    h *= np.uint32(0xBB67AE85)
    h ^= h >> np.uint32(16)
    return h


def _exact_adamw(s):
    t, (b1, b2) = s["step"] + 1, BETAS
    g, m, v = (s[k].double() for k in ("g", "m", "v"))
    if "ms" in s:
        m = m * s["ms"].double().repeat_interleave(BLOCK)
        v = v * s["vs"].double().repeat_interleave(BLOCK)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    hat = (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    out = {"p": s["p"].double() * (1 - LR * DECAY) - LR * hat, "m": m, "v": v}
    if "ms" not in s:
        return out
    with np.errstate(over="ignore"):
        at = np.uint32(0x9E3779B9) * np.arange(s["ms"].numel(), dtype=np.uint32)
        first = _hash32(np.array([t]) & 0xFFFFFFFF) ^ np.uint32(s["seed"])
        key = _hash32(at + _hash32(first))
        h = _hash32((key[:, None] + np.uint32(0x9E3779B9) * np.arange(BLOCK, dtype=np.uint32))
                    .reshape(-1))
    for name, x, u, top, bits, least in (("m", m, h & 0xFFFF, 7, 3, -6),
                                         ("v", v, h >> 16, 14, 2, -14)):
        u = torch.from_numpy(u.astype(np.int64)).to(x.device).double() / 65536
        most = x.abs().view(-1, BLOCK).amax(1)
        scale = torch.exp2((torch.frexp(most / math.sqrt(3))[1] - 1 - top).clamp(min=-126).double())
        scale = torch.where(most > 0, scale, 2.0 ** -126)
        a = x.abs() / scale.repeat_interleave(BLOCK)
        step = torch.exp2((torch.frexp(a)[1] - 1).clamp(min=least).double() - bits)
        q = torch.floor(a / step + u) * step
        if name == "v":
            q = torch.where(a > 0, q.clamp(min=2.0 ** -16), q)
        out[name], out[name + "s"] = q * torch.sign(x), scale
    return out
