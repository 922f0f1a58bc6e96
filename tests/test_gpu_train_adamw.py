"""adamw_step and optim.AdamW against the formula in 64 bits; the 8-bit codes
bit for bit against their definition (train_reference.states8)."""
import copy

import pytest
import torch

import train_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda"
SIZES = [1, 3, 4, 255, 256, 257, 1000, 4096, 4097, 20_001]
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)


def _inputs(sizes, dtype, seed, bits=32):
    gen = torch.Generator().manual_seed(seed)
    p = [torch.randn(n, generator=gen).to(dtype) for n in sizes]
    g = [(torch.randn(n, generator=gen) * torch.exp(torch.randn(n, generator=gen)) * 1e-2)
         .to(dtype) for n in sizes]
    m = [torch.randn(n, generator=gen) * 5e-3 for n in sizes]
    v = [torch.rand(n, generator=gen) * 1e-4 for n in sizes]
    if bits == 32:
        return p, g, m, v, None, None
    q = [R.states8(a, b, 7, 99, k) for k, (a, b) in enumerate(zip(m, v))]
    return (p, g, [x[0].to(torch.float8_e4m3fn) for x in q],
            [x[2].to(torch.float8_e5m2) for x in q], [x[1] for x in q], [x[3] for x in q])


def _held(code, scale):
    return (R.blocks_of(code.float()) * scale[:, None]).view(-1)[:code.numel()]


def _p_want(p, m, v, step, lr, betas, eps, weight_decay):
    """The new parameter in 64 bits from the new moments, and its bound: the
    quotient m / (sqrt(v) root + eps) is off by at most 16 units of 2^-24 (the
    moments 4, which weigh 1 and 1/2; root, square root, sum, reciprocal and
    product one or two each) where m's terms do not cancel, see _m_bound."""
    root = (1 - betas[1] ** step) ** -0.5
    upd = lr / (1 - betas[0] ** step) * m / (v.sqrt() * root + eps)
    return p * (1 - lr * weight_decay) - upd, upd


def _close_step(p1, p0, g, m0, v0, m1, v1, step, dtype, what, sign=1.0, **hy):
    p0, g, m0, v0 = (t.double() for t in (p0, g, m0, v0))
    b1, b2 = hy["betas"]
    g = g * sign
    m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
    u = 2.0 ** -24
    em = 4 * u * (b1 * m0.abs() + (1 - b1) * g.abs()) + 1e-44
    ev = 6 * u * v + 1e-44
    if m1 is not None:
        R.close(m1, (m, em), what + " m")
        R.close(v1, (v, ev), what + " v")
    want, upd = _p_want(p0, m, v, step, **hy)
    root = (1 - b2 ** step) ** -0.5
    e = (hy["lr"] / (1 - b1 ** step)) * em / (v.sqrt() * root + hy["eps"]) + 20 * u * upd.abs() \
        + 4 * u * p0.abs()
    R.close(p1, (want, e + R.HALF[dtype] * (want.abs() + e) + R.TINY[dtype]), what + " p")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("step", [1, 2, 1000])
@pytest.mark.parametrize("maximize", [False, True])
def test_states_in_32_bits(step, maximize, dtype):
    from fedsim_amd.train_ops import adamw_step

    p, g, m, v, _, _ = _inputs(SIZES, dtype, step)
    dev = [[t.to(DEV) for t in ts] for ts in (p, g, m, v)]
    adamw_step(*dev, step=step, maximize=maximize, **HYPER)
    for k, n in enumerate(SIZES):
        assert torch.equal(dev[1][k].cpu(), g[k])
        _close_step(dev[0][k], p[k], g[k], m[k], v[k], dev[2][k], dev[3][k], step, dtype, str(n),
                    -1.0 if maximize else 1.0, **HYPER)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("step", [1, 50])
def test_states_in_8_bits(step, dtype):
    from fedsim_amd.train_ops import adamw_step

    p, g, m, v, ms, vs = _inputs(SIZES, dtype, step + 5, 8)
    dev = [[t.to(DEV) for t in ts] for ts in (p, g, m, v, ms, vs)]
    adamw_step(*dev, step=step, seed=77, **HYPER)
    block = 0
    for k, n in enumerate(SIZES):
        m0, v0 = _held(m[k], ms[k]), _held(v[k], vs[k])
        m1, v1 = R.moments32(m0, v0, g[k].float(), HYPER["betas"])
        qm, sm, qv, sv = R.states8(m1, v1, step, 77, block)
        block += -(-n // R.BLOCK)
        assert torch.equal(dev[4][k].cpu(), sm) and torch.equal(dev[5][k].cpu(), sv), n
        assert torch.equal(dev[2][k].float().cpu(), qm), n
        assert torch.equal(dev[3][k].float().cpu(), qv), n
        _close_step(dev[0][k], p[k], g[k], m0, v0, None, None, step, dtype, str(n), **HYPER)


def test_rounding_is_unbiased():
    """One value at 40 places of each of 4096 blocks, whose mean after rounding
    is its own: the mean of n = 163 840 roundings with spacing s has a standard
    deviation of at most s / (2 sqrt n); six of them are allowed."""
    from fedsim_amd.train_ops import adamw_step

    blocks = 4096
    n = blocks * R.BLOCK
    for x in (0.7123, 0.0301, 1.3e-4, 3.3e-6):
        m0 = torch.zeros(blocks, R.BLOCK)
        m0[:, 0] = 1.0  # sets the scale: 2^-7 steps of 2^-3 below it
        m0[:, 1:41] = x
        v0 = m0.clone()
        m1, v1 = R.moments32(m0, v0, torch.zeros(blocks, R.BLOCK), (0.0, 0.0))
        # betas of 0 and a gradient: m = g, v = g g
        g = m0.view(-1).to(DEV)
        p = torch.zeros(n, device=DEV)
        em, ev = torch.zeros(n, device=DEV).to(torch.float8_e4m3fn), \
            torch.zeros(n, device=DEV).to(torch.float8_e5m2)
        sm, sv = torch.ones(blocks, device=DEV), torch.ones(blocks, device=DEV)
        adamw_step([p], [g], [em], [ev], [sm], [sv], step=1, lr=0.0, betas=(0.0, 0.0), seed=5)
        for code, scale, want, mant, least in ((em, sm, x, 3, 2.0 ** -9),
                                               (ev, sv, x * x, 2, 2.0 ** -16)):
            s = float(scale[0])
            got = (code.float().view(blocks, R.BLOCK)[:, 1:41] * s).double()
            spacing = max(least * s, want * 2.0 ** -mant)
            if code is ev and want < least * s:
                assert bool((got == least * s).all())  # never rounded to zero
                continue
            lo, hi = float(got.min()), float(got.max())
            assert lo <= want <= hi and hi - lo <= spacing * 1.001, (x, lo, hi, want)
            assert abs(float(got.mean()) - want) < 6 * spacing / 2 / (blocks * 40) ** 0.5, x


def test_moments_in_8_bits_follow_a_change():
    """Rounding to nearest would leave v in place: with b2 = 0.999 a step moves
    it by less than half a code's spacing.  500 steps of a gradient twice as
    large take v to 4 - 3 * 0.999^500 = 2.18 times its value in the mean; 8 192
    elements whose relative deviation is below 1 give a mean within 6 / sqrt(8192)
    = 0.07 of that, relative."""
    from fedsim_amd.train_ops import adamw_step

    n = 8192
    p, g = torch.zeros(n, device=DEV), torch.full((n,), 2.0, device=DEV)
    m, v = torch.zeros(n), torch.ones(n)
    q = R.states8(m, v, 1, 0)
    em, ev = q[0].to(torch.float8_e4m3fn).to(DEV), q[2].to(torch.float8_e5m2).to(DEV)
    sm, sv = q[1].to(DEV), q[3].to(DEV)
    first = float(_held(ev.cpu(), sv.cpu()).mean())
    for t in range(500):
        adamw_step([p], [g], [em], [ev], [sm], [sv], step=t + 1, lr=0.0, betas=(0.9, 0.999))
    want = 4 - (4 - first) * 0.999 ** 500
    got = float(_held(ev.cpu(), sv.cpu()).mean())
    assert abs(got / want - 1) < 0.07, (got, want)


def test_infinities_and_nan_are_that_elements_alone():
    from fedsim_amd.train_ops import adamw_step

    n = 700
    for bits in (32, 8):
        p, g, m, v, ms, vs = _inputs([n], torch.float32, 3, bits)
        clean = [[t.to(DEV) for t in ts] for ts in (p, g, m, v)] + \
            ([[t.to(DEV) for t in ts] for ts in (ms, vs)] if bits == 8 else [])
        bad = [[t.clone() for t in ts] for ts in clean]
        bad[1][0][5], bad[1][0][300], bad[1][0][301] = float("nan"), float("inf"), float("-inf")
        for x in (clean, bad):
            adamw_step(*x, step=3, **HYPER)
        hit = torch.zeros(n, dtype=torch.bool)
        hit[[5, 300, 301]] = True
        ok = [k for k in range(n) if not hit[k]]
        for k in (0, 2, 3):
            a, b = clean[k][0].float().cpu(), bad[k][0].float().cpu()
            # another largest element may have set the block's scale
            if bits == 32 or k == 0:
                assert torch.equal(a[ok], b[ok])
            assert b[ok].isfinite().all()
        assert bad[0][0][5].isnan() and bad[2][0].float()[5].isnan()
        assert not bad[2][0].float()[[300, 301]].isfinite().any()
        assert bad[3][0].float()[5].isnan() and (bad[3][0].float()[[300, 301]]
                                                 == float("inf")).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_whose_squares_are_subnormal(bits):
    """The first step is -lr sign(g) however small g is, with eps = 0.  v = 1e-2 g^2
    of 1e-42 and more has 714 units of 2^-149 and is off by one: 0.0015, half of it
    in the root."""
    from fedsim_amd.optim import AdamW

    g = torch.tensor([1e-20, -1e-20, 3e-20, 1e-19, -1e-17, 1e-12] * 100)
    p = torch.nn.Parameter(torch.zeros(600, device=DEV))
    p.grad = g.to(DEV)
    AdamW([p], lr=0.5, betas=(0.9, 0.99), eps=0.0, weight_decay=0.0, state_bits=bits).step()
    off = (p.detach().cpu() + 0.5 * torch.sign(g)).abs().max()
    assert float(off) < 0.5 * (0.5 / 714 + 32 * 2.0 ** -24)


def test_many_tensors_offsets_and_neighbours():
    """150 tensors of all alignments inside one buffer: more than a launch
    takes; what lies between them stays as it was."""
    from fedsim_amd.train_ops import adamw_step

    gen = torch.Generator().manual_seed(8)
    sizes = [int(x) for x in torch.randint(1, 900, (150,), generator=gen)]
    total = sum(n + 3 for n in sizes)
    for dtype in DTYPES:
        flat = [torch.rand(total, generator=gen).to(dtype).to(DEV) for _ in range(2)] + \
            [torch.rand(total, generator=gen).to(DEV) for _ in range(2)]
        before = [f.cpu().clone() for f in flat]
        views, at = [[] for _ in flat], 1
        inside = torch.zeros(total, dtype=torch.bool)
        for n in sizes:
            inside[at:at + n] = True
            for f, vs in zip(flat, views):
                vs.append(f[at:at + n])
            at += n + 3
        adamw_step(*views, step=4, **HYPER)
        at = [f.cpu() for f in flat]
        for a, b in zip(at, before):
            assert torch.equal(a[~inside], b[~inside])
        _close_step(at[0][inside], *(b[inside] for b in before), at[2][inside], at[3][inside], 4,
                    dtype, str(dtype), **HYPER)


def _model(dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(40, 33), torch.nn.ReLU(),
                               torch.nn.Linear(33, 5)).to(DEV).to(dtype)


def _train(model, opt, steps, seed=0):
    gen = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        x = torch.randn(16, 40, generator=gen).to(DEV).to(next(model.parameters()).dtype)
        model(x).square().mean().backward()
        opt.step()
        opt.zero_grad()


def test_optimizer_follows_torchs():
    """20 steps on gradients that both get: each step is off by at most 24
    units of 2^-24 of |p| + lr."""
    from fedsim_amd.optim import AdamW

    a = [torch.nn.Parameter(t.to(DEV)) for t in _inputs([1000, 33], torch.float32, 1)[0]]
    b = [torch.nn.Parameter(t.detach().double().cpu()) for t in a]
    ours = AdamW(a, lr=1e-2, weight_decay=0.1)
    theirs = torch.optim.AdamW(b, lr=1e-2, weight_decay=0.1)
    gen = torch.Generator().manual_seed(1)
    for k in range(20):
        for p, q in zip(a, b):
            if k == 3 and p.numel() == 33:
                p.grad = q.grad = None  # that parameter's step is left out
                continue
            g = torch.randn(p.shape, generator=gen)
            p.grad, q.grad = g.to(DEV), g.double()
        ours.step()
        theirs.step()
    assert [ours.state[p]["step"] for p in a] == [20, 19]
    for p, q in zip(a, b):
        R.close(p, (q.detach(), 20 * 24 * 2.0 ** -24 * (q.detach().abs() + 0.3)), "p")


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_state_dict_goes_on_where_it_was(bits, capturable, dtype):
    from fedsim_amd.optim import AdamW

    kw = dict(lr=1e-2, state_bits=bits, seed=3, capturable=capturable)
    one = _model(dtype)
    opt = AdamW(one.parameters(), **kw)
    _train(one, opt, 3)
    two = copy.deepcopy(one)
    opt2 = AdamW(two.parameters(), **kw)
    saved = copy.deepcopy(opt.state_dict())
    opt2.load_state_dict(saved)
    _train(one, opt, 3, 1)
    _train(two, opt2, 3, 1)
    for p, q in zip(one.parameters(), two.parameters()):
        assert torch.equal(p, q)
        s, t = opt.state[p], opt2.state[q]
        assert int(s["step"]) == int(t["step"]) == 6
        for k in s:
            if isinstance(s[k], torch.Tensor) and k != "step":
                assert s[k].dtype == t[k].dtype and torch.equal(s[k].float(), t[k].float()), k
    # the groups' options are the saved ones
    three = copy.deepcopy(two)
    opt3 = AdamW(three.parameters(), state_bits=40 - bits)
    opt3.load_state_dict(opt2.state_dict())
    assert opt3.param_groups[0]["state_bits"] == bits
    _train(two, opt2, 2, 2)
    _train(three, opt3, 2, 2)
    assert all(torch.equal(p, q) for p, q in zip(two.parameters(), three.parameters()))


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_step_counts_on(bits):
    """A replayed graph takes the steps that eager calls take, bit for bit."""
    from fedsim_amd.optim import AdamW

    pair = []
    for _ in range(2):
        ps = [torch.nn.Parameter(t.to(DEV)) for t in _inputs([1000, 33, 257], torch.float32, 1)[0]]
        for p in ps:
            p.grad = torch.ones_like(p)
        opt = AdamW(ps, lr=1e-2, state_bits=bits, capturable=True, seed=9)
        opt.step()
        pair.append((ps, opt))
    (a, oa), (b, ob) = pair
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        oa.step()
    gen = torch.Generator().manual_seed(2)
    for _ in range(4):
        for p, q in zip(a, b):
            new = torch.randn(p.shape, generator=gen).to(DEV)
            p.grad.copy_(new)
            q.grad.copy_(new)
        g.replay()
        ob.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            assert int(oa.state[p]["step"]) == int(ob.state[q]["step"])
            for k in ("exp_avg", "exp_avg_sq"):
                assert torch.equal(oa.state[p][k].float(), ob.state[q][k].float())
    assert int(oa.state[a[0]]["step"]) == 5


def test_capture_refusals():
    from fedsim_amd.optim import AdamW

    for capturable, steps, message in ((False, 1, "capturable"), (True, 0, "before capturing")):
        p = torch.nn.Parameter(torch.ones(10, device=DEV))
        p.grad = torch.ones_like(p)
        opt = AdamW([p], capturable=capturable)
        for _ in range(steps):
            opt.step()
        g = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=message):
            with torch.cuda.graph(g):
                opt.step()
    torch.cuda.synchronize()
    opt.step()


def test_a_loaded_state_takes_a_step_before_a_capture():
    """A loaded state's step is the host's number: a graph that put it on the
    device would start from it at every replay."""
    from fedsim_amd.optim import AdamW

    p = torch.nn.Parameter(torch.ones(10, device=DEV))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], capturable=True)
    opt.step()
    opt.load_state_dict(opt.state_dict())
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    for k in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert int(opt.state[p]["step"]) == 3 + k


def test_same_bits_every_time_and_on_another_stream():
    from fedsim_amd.train_ops import adamw_step

    results = []
    side = torch.cuda.Stream()
    for k in range(3):
        args = [[t.to(DEV) for t in ts] for ts in _inputs(SIZES, torch.bfloat16, 4, 8)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side if k == 1 else torch.cuda.current_stream()):
            adamw_step(*args, step=6, seed=1, **HYPER)
        torch.cuda.synchronize()
        results.append([t.float().cpu() for ts in args for t in ts])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_a_round_with_adamw_on_clients_and_server():
    """One FedAvg server step with AdamW as its optimizer: the averaged
    pseudo-gradient goes through the same kernel."""
    from fedsim_amd.distributed.centralized.training import FedAvg
    from fedsim_amd.optim import AdamW
    from fedsim_amd.utils import SerialAggregator, Storage

    P = 4099
    gen = torch.Generator().manual_seed(6)
    rows = torch.randn(3, P, generator=gen)
    cloud0 = torch.randn(P, generator=gen)
    for bits in (32, 8):
        cloud = cloud0.to(DEV).requires_grad_(True)
        st, agg = Storage(), SerialAggregator()
        opt = AdamW([cloud], lr=0.1, state_bits=bits)
        for key, val in (("cloud_params", cloud), ("optimizer", opt), ("lr_scheduler", None)):
            st.write(key, val)
        for k in range(3):
            msg = dict(local_params=rows[k].to(DEV), num_steps=1, diverged=False,
                       num_samples={"train": 2 + k}, metrics={"train": {}})
            assert FedAvg.receive_from_client(st, k, msg, "train", agg, None)
        FedAvg.optimize(st, agg, None)
        w = torch.tensor([2., 3., 4.], dtype=torch.float64)[:, None]
        g = cloud0.double() - (rows.double() * w).sum(0) / 9
        want = cloud0.double() * (1 - 0.1 * 0.01) - 0.1 * g / (g.abs() + 1e-8)
        # the gradient is off by 2^-21 at most; the step's sign(g) is as good as
        # g where |g| stands above that
        sure = g.abs() > 1e-3
        off = (cloud.detach().cpu().double() - want).abs()[sure]
        assert float(off.max()) < 1e-5 and int(opt.state[cloud]["step"]) == 1
