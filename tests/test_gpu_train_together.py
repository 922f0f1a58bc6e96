"""The training operators as a run: a cohort of client models in the rows of one
slab takes a step (grouped_linear twice, the loss's gradient, AdamW) and is
averaged; one client trains by local_train; a captured step goes on where the
eager one stopped."""
import pytest
import torch

import train_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
I, H, O = 84, 40, 10
SIZES = [(H, I), (H,), (O, H), (O,)]
P = sum(torch.Size(s).numel() for s in SIZES)


def _layers(slab):
    """W1, b1, W2, b2 of the models in the slab's rows, as views."""
    out, at = [], 0
    for s in SIZES:
        n = torch.Size(s).numel()
        out.append(slab[:, at:at + n].unflatten(1, s))
        at += n
    return out


def _cohort(edges, seed=0):
    gen = torch.Generator().manual_seed(seed)
    G, N = len(edges) - 1, edges[-1]
    slab = torch.randn(G, P, generator=gen) * 0.15
    return slab, torch.randn(N, I, generator=gen), torch.randint(0, O, (N,), generator=gen)


def _loss(slab, x, y, offsets, scale):
    from fedsim_amd.functional import grouped_linear

    w1, b1, w2, b2 = _layers(slab)
    h = grouped_linear(x, w1, offsets, b1, activation="relu")
    z = grouped_linear(h, w2, offsets, b2)
    return (torch.nn.functional.cross_entropy(z, y, reduction="none") * scale).sum()


def _gradient64(slab, x, y, edges, scale):
    """The slab's gradient by the formulas, and a bound of the float32 run's
    distance from it: each product's own bound (R.product), and the bounds of its
    operands carried through it."""
    slab, x, scale = slab.double(), x.double(), scale.double()
    w1, b1, w2, b2 = _layers(slab)
    f = torch.float32
    h, eh = R.product(x, w1, b1, None, "relu", f, None, edges)["y"]
    z, ez = R.product(h, w2, b2, None, "none", f, None, edges)["y"]
    for g in range(len(edges) - 1):
        s = slice(edges[g], edges[g + 1])
        ez[s] += eh[s] @ w2[g].abs().T
    p = torch.softmax(z, 1)
    d = (p - torch.nn.functional.one_hot(y, O)) * scale[:, None]
    # a softmax moves by at most twice its logits' largest error; float32's own
    # exponentials and sums of 10 by less than 32 roundings
    ed = (2 * ez.amax(1, keepdim=True) + 32 * 2.0 ** -24).expand_as(d) * scale[:, None]
    two = R.product(h, w2, b2, None, "none", f, d, edges)
    dh, edh = two["dx"]
    for g in range(len(edges) - 1):
        s = slice(edges[g], edges[g + 1])
        two["dw"][1][g] += ed[s].T @ (h[s].abs() + eh[s]) + d[s].abs().T @ eh[s]
        two["db"][1][g] += ed[s].sum(0)
        edh[s] += ed[s] @ w2[g].abs()
    one = R.product(x, w1, b1, None, "relu", f, dh, edges)
    for g in range(len(edges) - 1):
        s = slice(edges[g], edges[g + 1])
        one["dw"][1][g] += edh[s].T @ x[s].abs()
        one["db"][1][g] += edh[s].sum(0)
    return tuple(torch.cat([t[k].flatten(1) for t in (one["dw"], one["db"], two["dw"], two["db"])],
                           1) for k in (0, 1))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_cohort_steps_and_is_averaged(bits):
    from fedsim_amd.optim import AdamW
    from fedsim_amd.utils import SerialAggregator

    edges = [0, 37, 37, 38, 170, 300]
    counts = torch.tensor([b - a for a, b in zip(edges, edges[1:])])
    slab0, x, y = _cohort(edges)
    scale = torch.repeat_interleave(1.0 / counts.clamp(min=1), counts)
    g, eg = _gradient64(slab0, x, y, edges, scale)

    slab = torch.nn.Parameter(slab0.to(DEV))
    lr, eps = 0.02, 0.01
    opt = AdamW([slab], lr=lr, eps=eps, weight_decay=0.1, state_bits=bits)
    off = torch.tensor(edges, device=DEV)
    _loss(slab, x.to(DEV), y.to(DEV), off, scale.to(DEV)).backward()
    R.close(slab.grad, (g, eg), "gradient")
    assert not slab.grad[1].any()  # the client without a sample
    opt.step()

    # the first step is -lr g / (|g| + eps), of slope lr / eps at most; its
    # float32 arithmetic takes fewer than 16 roundings of the step and of p
    want = slab0.double() * (1 - lr * 0.1) - lr * g / (g.abs() + eps)
    bound = lr / eps * eg + 16 * 2.0 ** -24 * (lr + want.abs())
    R.close(slab, (want, bound), "parameters")

    agg = SerialAggregator()
    for k in (0, 2, 3, 4):
        agg.add("local_params", slab.detach()[k], int(counts[k]))
    got = agg.pop("local_params")
    w = counts.double()[:, None]
    mean = (want * w).sum(0) / w.sum()
    e = ((bound + 8 * 2.0 ** -24 * want.abs()) * w).sum(0) / w.sum()
    R.close(got, (mean, e), "average")


class _Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.a = torch.nn.Linear(I, H)
        self.b = torch.nn.Linear(H, O)

    def forward(self, x):
        from fedsim_amd.functional import linear_act

        h = linear_act(x, self.a.weight, self.a.bias, activation="gelu")
        return linear_act(h, self.b.weight, self.b.bias)


@pytest.mark.parametrize("bits", [32, 8])
def test_local_train_with_adamw(bits):
    """A client's own loop: finite, counted, and the same bits when run again."""
    from functools import partial

    from fedsim_amd.local import local_train
    from fedsim_amd.optim import AdamW
    from fedsim_amd.scores import CrossEntropyScore

    gen = torch.Generator().manual_seed(3)
    data = [(torch.randn(n, I, generator=gen), torch.randint(0, O, (n,), generator=gen))
            for n in (32, 32, 1)]
    runs = []
    for _ in range(2):
        torch.manual_seed(1)
        net = _Net().to(DEV)
        start = [p.detach().clone() for p in net.parameters()]
        opt = partial(AdamW, lr=1e-2, state_bits=bits)(net.parameters())
        assert local_train(net, data, 2, 0, CrossEntropyScore(), opt, device=DEV) == (130, 6, False)
        now = [p.detach().clone() for p in net.parameters()]
        assert all(t.isfinite().all() and not torch.equal(t, s) for t, s in zip(now, start))
        assert all(opt.state[p]["step"] == 6 for p in net.parameters())
        runs.append(now)
    # torch's own share of the step (its loss, its clipping) is repeatable too
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_goes_on_where_the_eager_one_stopped(bits):
    """Forward, backward and AdamW in one graph: every replay gives the eager
    run's bits, with the rows of the groups changed between replays."""
    from fedsim_amd.optim import AdamW

    edges = [0, 37, 37, 38, 170, 300]
    slab0, x0, y0 = _cohort(edges, 5)
    scale = torch.full((300,), 0.01, device=DEV)
    a = torch.nn.Parameter(slab0.to(DEV))
    b = torch.nn.Parameter(slab0.to(DEV))
    x, y = x0.to(DEV), y0.to(DEV)
    off = torch.tensor(edges, device=DEV)
    oa = AdamW([a], lr=1e-2, state_bits=bits, capturable=True)
    ob = AdamW([b], lr=1e-2, state_bits=bits)

    def step(p, opt):
        p.grad.zero_()
        _loss(p, x, y, off, scale).backward()
        opt.step()

    a.grad, b.grad = torch.zeros_like(a), torch.zeros_like(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, oa)
    torch.cuda.current_stream().wait_stream(side)
    step(b, ob)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(a, oa)
    gen = torch.Generator().manual_seed(8)
    for k in range(4):
        x.copy_(torch.randn(x.shape, generator=gen))
        off.copy_(torch.tensor([0, 10 * k, 10 * k, 100, 299 - k, 300 - k]))
        g.replay()
        step(b, ob)
        torch.cuda.synchronize()
        assert torch.equal(a.grad, b.grad) and torch.equal(a, b), k
    assert int(oa.state[a]["step"]) == 5
