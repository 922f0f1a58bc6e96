"""optim.AdamW beyond its plain loop: parameters that join late or sit a step
out, steps that fail, states of other optimizers; and adamw_step's refusals of
shared memory."""
import copy

import pytest
import torch

import train_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _pair(sizes, seed, **kw):
    """Ours on the device and torch's in 64 bits, from the same values."""
    from fedsim_amd.optim import AdamW

    gen = torch.Generator().manual_seed(seed)
    a = [torch.nn.Parameter(torch.randn(n, generator=gen).to(DEV)) for n in sizes]
    b = [torch.nn.Parameter(t.detach().double().cpu()) for t in a]
    hy = dict(lr=1e-2, weight_decay=0.1)
    return gen, a, b, AdamW(a, **hy, **kw), torch.optim.AdamW(b, **hy)


def _grads(gen, a, b, without=()):
    for k, (p, q) in enumerate(zip(a, b)):
        g = torch.randn(p.shape, generator=gen)
        if k in without:
            p.grad = q.grad = None
        else:
            p.grad, q.grad = g.to(DEV), g.double()


def _same(a, b, steps):
    # 24 units of 2^-24 of |p| + lr a step, as where no step is left out
    for p, q in zip(a, b):
        R.close(p, (q.detach(), steps * 24 * 2.0 ** -24 * (q.detach().abs() + 0.3)), "p")


@pytest.mark.parametrize("capturable", [False, True])
def test_each_parameter_counts_its_own_steps(capturable):
    """One skips a step, one gets its first gradient late: both have their own
    bias correction, as torch's."""
    gen, a, b, ours, theirs = _pair([1000, 33, 300], 1, capturable=capturable)
    for k in range(20):
        without = ({1} if k in (3, 9) else set()) | ({2} if k < 12 else set())
        _grads(gen, a, b, without)
        ours.step()
        theirs.step()
    assert [int(ours.state[p]["step"]) for p in a] == [20, 18, 8]
    _same(a, b, 20)


@pytest.mark.parametrize("capturable", [False, True])
def test_loaded_counts_stay_apart(capturable):
    """Counts that differ in a saved state differ after it is loaded, whichever
    way they were counted before."""
    from fedsim_amd.optim import AdamW

    for saved_as in (False, True):
        gen, a, b, ours, theirs = _pair([257, 40], 2, capturable=saved_as)
        for k in range(6):
            _grads(gen, a, b, {1} if k < 4 else ())
            ours.step()
            theirs.step()
        saved = copy.deepcopy(ours.state_dict())
        saved["param_groups"][0]["capturable"] = capturable
        two = [torch.nn.Parameter(p.detach().clone()) for p in a]
        opt = AdamW(two, capturable=capturable)
        opt.load_state_dict(saved)
        for _ in range(3):
            _grads(gen, two, b)
            opt.step()
            theirs.step()
        assert [int(opt.state[p]["step"]) for p in two] == [9, 5]
        _same(two, b, 9)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_of_different_counts(bits):
    """A graph of some parameters' step, with eager steps of others between its
    replays: the counts, and so the bits, are those of the run without a graph."""
    runs = []
    for graphed in (True, False):
        gen, a, b, opt, _ = _pair([1000, 33, 700], 3, capturable=True, state_bits=bits)

        def fill(k):
            for p in a:
                g = torch.randn(p.shape, generator=gen).to(DEV)
                if p.grad is None:
                    p.grad = g
                else:
                    p.grad.copy_(g)

        fill(0)
        late, a[2].grad = a[2].grad, None
        opt.step()  # the first two
        a[2].grad = late
        opt.step()  # all: counts 2, 2, 1
        if graphed:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
        for k in range(4):
            fill(k)
            if graphed:
                graph.replay()
            else:
                opt.step()
            kept, a[0].grad = a[0].grad, None
            opt.step()  # the last two
            a[0].grad = kept
            torch.cuda.synchronize()
        assert [int(opt.state[p]["step"]) for p in a] == [6, 10, 9]
        runs.append([p.detach().clone() for p in a])
    assert all(torch.equal(p, q) for p, q in zip(*runs))


def test_many_counted_steps_on_the_device():
    """More tensors than one launch takes, each with a count of its own, give the
    bits of a call with that step for each."""
    from fedsim_amd.train_ops import adamw_step

    gen = torch.Generator().manual_seed(4)
    sizes = [int(n) for n in torch.randint(1, 900, (130,), generator=gen)]
    for bits in (32, 8):
        def fresh():
            g = torch.Generator().manual_seed(5)
            p = [torch.randn(n, generator=g).to(DEV) for n in sizes]
            d = [torch.randn(n, generator=g).to(DEV) for n in sizes]
            blocks = [-(-n // 256) for n in sizes]
            if bits == 32:
                return [p, d, [torch.zeros_like(t) for t in p], [torch.zeros_like(t) for t in p]]
            return [p, d, [torch.zeros(n, device=DEV).to(torch.float8_e4m3fn) for n in sizes],
                    [torch.zeros(n, device=DEV).to(torch.float8_e5m2) for n in sizes],
                    [torch.ones(k, device=DEV) for k in blocks],
                    [torch.ones(k, device=DEV) for k in blocks]]

        one, two = fresh(), fresh()
        counts = [1 + k * k % 97 for k in range(len(sizes))]
        first = [sum(-(-m // 256) for m in sizes[:k]) for k in range(len(sizes))]
        adamw_step(*one, step=[torch.tensor([c], device=DEV) for c in counts], lr=1e-2, seed=7)
        for k, c in enumerate(counts):
            adamw_step(*[ts[k:k + 1] for ts in two], step=c, lr=1e-2, seed=7,
                       first_blocks=first[k:k + 1])
        for s, t in zip(one, two):
            for k, (u, v) in enumerate(zip(s, t)):
                assert torch.equal(u.float(), v.float()), (bits, k)
    bad = fresh()
    one = torch.ones(1, dtype=torch.int64, device=DEV)
    for step in ([one] * 129, [one] * 129 + [one.float()], [one] * 129 + [one.cpu()],
                 [one] * 129 + [one.expand(2)], [one] * 129 + [1]):
        with pytest.raises((ValueError, TypeError)):
            adamw_step(*bad, step=step, lr=1e-2)


@pytest.mark.parametrize("capturable", [False, True])
def test_a_step_that_raises_is_not_counted(capturable):
    """A gradient of another size than its parameter's (a parameter resized
    through .data), mended: the next step is the second."""
    gen, a, b, ours, theirs = _pair([64, 10], 6, capturable=capturable)
    _grads(gen, a, b)
    ours.step()
    theirs.step()
    _grads(gen, a, b)
    whole = a[1].data
    a[1].data = torch.zeros(11, device=DEV)
    with pytest.raises(ValueError):
        ours.step()
    a[1].data = whole
    assert [int(ours.state[p]["step"]) for p in a] == [1, 1]
    ours.step()
    theirs.step()
    assert [int(ours.state[p]["step"]) for p in a] == [2, 2]
    _same(a, b, 2)


def test_an_epsilon_below_the_smallest_normal_number():
    """m = 0 and v = 0 over eps: no change, for every eps above 0."""
    from fedsim_amd.train_ops import adamw_step

    for eps in (1e-30, 1e-39, 1e-45, 1e-60):
        p, g = torch.full((300,), 2.0, device=DEV), torch.zeros(300, device=DEV)
        g[7] = 1.0
        m, v = torch.zeros(300, device=DEV), torch.zeros(300, device=DEV)
        adamw_step([p], [g], [m], [v], step=1, lr=0.5, eps=eps, weight_decay=0.0)
        assert abs(float(p[7]) - 1.5) < 32 * 2.0 ** -24
        p[7] = 2.0
        assert (p == 2.0).all(), eps


def test_a_state_of_torchs_adamw():
    """Its options lack this class's own, which stay as they were given; what
    this class does not have is refused."""
    from fedsim_amd.optim import AdamW

    gen = torch.Generator().manual_seed(8)
    b = [torch.nn.Parameter(torch.randn(n, generator=gen)) for n in (100, 33)]
    theirs = torch.optim.AdamW(b, lr=1e-2, weight_decay=0.1)
    for _ in range(3):
        for q in b:
            q.grad = torch.randn(q.shape, generator=gen)
        theirs.step()
    two = [torch.nn.Parameter(q.detach().to(DEV)) for q in b]
    opt = AdamW(two, seed=5)
    opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["state_bits"] == 32 and opt.param_groups[0]["seed"] == 5
    for p, q in zip(two, b):
        q.grad = torch.randn(q.shape, generator=gen)
        p.grad = q.grad.to(DEV)
    opt.step()
    theirs.step()
    assert [int(opt.state[p]["step"]) for p in two] == [4, 4]
    for p, q in zip(two, b):  # a step each in float32
        q = q.detach().double()
        R.close(p, (q, 2 * 24 * 2.0 ** -24 * (q.abs() + 0.3)), "p")
    with pytest.raises(ValueError, match="state_bits"):
        AdamW(two, state_bits=8).load_state_dict(theirs.state_dict())
    saved = torch.optim.AdamW(b, amsgrad=True).state_dict()
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(saved)
    assert not opt.param_groups[0].get("amsgrad")


def test_what_a_step_writes_shares_no_memory():
    """Each list against each other one; gradients may share among themselves."""
    from fedsim_amd.train_ops import adamw_step

    f8, f8v = torch.float8_e4m3fn, torch.float8_e5m2

    def f32(n=300):
        return torch.ones(n, device=DEV)

    hy = dict(step=1, lr=1e-3)
    p = f32()
    two = f32(600)
    for bad in ([p, p, f32(), f32()], [p, f32(), p, f32()], [p, f32(), f32(), p],
                [f32(), p, p, f32()], [f32(), p, f32(), p], [f32(), f32(), p, p],
                [two[:300], two[200:500], f32(), f32()],  # a gradient at an offset
                [two[200:500], two[:300], f32(), f32()],
                [two[:300], f32(), two[299:599], f32()],
                [f32(), f32(), two[299:599], two[:300]]):
        with pytest.raises(ValueError, match="share memory"):
            adamw_step(*[[t] for t in bad], **hy)

    def eight():
        return [f32(), f32(), f32().to(f8), f32().to(f8v), f32(2), f32(2)]

    one = eight()
    raw = torch.zeros(600, dtype=torch.uint8, device=DEV)
    for k, t in ((5, one[4]), (4, one[0][:2]), (5, one[0][298:]), (5, one[1][:2]),
                 (2, raw[:300].view(f8)), (2, one[0].view(torch.uint8)[:300].view(f8))):
        bad = list(one)
        bad[k] = t
        if t.dtype == f8 and t.data_ptr() == raw.data_ptr():
            bad[3] = raw[100:400].view(f8v)
        with pytest.raises(ValueError, match="share memory"):
            adamw_step(*[[t] for t in bad], **hy)
    # a long range behind which short ones lie: the furthest counts
    slab = f32(1000)
    with pytest.raises(ValueError, match="share memory"):
        adamw_step([slab[:900], slab[950:]], [f32(900), f32(50)], [f32(900), f32(50)],
                   [f32(900), slab[800:850]], **hy)
    assert (two == 1).all() and (slab == 1).all() and (p == 1).all()
    g = f32(600)
    a, b = f32(), f32()
    adamw_step([a, b], [g[:300], g[100:400]], [torch.zeros_like(a) for _ in range(2)],
               [torch.zeros_like(a) for _ in range(2)], **hy)
    assert torch.equal(a, b) and (a < 1).all()
    # neighbours in one buffer share nothing
    slab = torch.rand(1200, device=DEV)
    adamw_step(*[[slab[k * 300:(k + 1) * 300]] for k in range(4)], **hy)
