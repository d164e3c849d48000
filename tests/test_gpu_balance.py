"""The router's balance loss and its gradient (``experts.balance_loss``) against the formula in 64 bits.

Bounds, u = 2^-24.  A probability is a power (2 units of 2^-23, and where results are of 16 bits or sums are made of it, its argument's rounding: d * 2^-24 of it for a
logit d below the largest) over a sum of n of them in a fixed tree: R(d) = (8 + n / 32 + 5 + d) * 2 u.  Sums over tokens add one u a token of a warp and the
trees of warps and CTAs."""
import numpy as np
import pytest
import torch

from flexspmv_b200 import experts
from flexspmv_b200.binding import FlexSpmvError

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24, torch.float32: 1e-37}


def logits_of(seed, tokens, n, dtype, masked=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = (torch.randn((tokens, n), generator=g, device="cuda") * 1.5 + torch.randn(n, generator=g, device="cuda")).to(dtype)
    if masked and tokens > 5:
        l[1] = float("-inf")                                                 # no token
        l[2, 1:] = float("-inf")
        l[3] = torch.finfo(dtype).min                                        # all alike
        l[4, : n // 2] = torch.finfo(dtype).min
        l[5, ::3] = float("-inf")
    return l


def softmax(l):
    """(probabilities, rows that are there, distance below the largest)"""
    l = l.double()
    there = (l > float("-inf")).any(1)
    top = torch.where(there, l.max(1).values, 0.0)[:, None]
    p = torch.exp(l - top)
    return p / torch.where(there, p.sum(1), 1.0)[:, None], there, torch.where(l > float("-inf"), top - l, 0.0).clamp(max=110)


def bound_of(p, d, n):
    return (13 + n / 32 + d) * 2 * U * p


def check_loss(b, l, plan):
    n = l.shape[1]
    p, there, d = softmax(l)
    counts = plan.offsets.diff()
    assert torch.equal(b.counts, counts) and int(b.tokens) == int(there.sum())
    t, pairs = max(1, int(there.sum())), max(1, int(counts.sum()))
    tree = (l.shape[0] / 148 / 8 + 1 + 16 + 148 + 4) * U
    mean = p.sum(0) / t
    em = (bound_of(p, d, n).sum(0) + (tree + 2 * U) * p.sum(0)) / t + 1e-37
    assert bool(((b.mean.double() - mean).abs() <= em).all())
    loss = float((mean * counts).sum()) * n / pairs
    assert abs(float(b.loss.double()) - loss) <= (float((em * counts).sum()) * n / pairs + (n / 32 + 40) * U * loss)


SIZES = [(0, 8, 2), (1, 1, 1), (1, 64, 8), (7, 60, 4), (64, 33, 6), (65, 8, 8), (333, 256, 8), (1000, 40, 1), (5001, 384, 7), (20011, 128, 2), (513, 1024, 32),
         (300, 500, 4), (90, 516, 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,n,k", SIZES)
def test_balance_loss(tokens, n, k, dtype):
    l = logits_of(tokens + n, tokens, n, dtype)
    plan = experts.route(l, k)
    b = experts.balance_loss(l, plan)
    check_loss(b, l, plan)
    again = experts.balance_loss(l, plan)
    assert all(torch.equal(x, y) for x, y in zip(b, again))
    room = torch.full((tokens, n + 3), float("nan"), dtype=dtype, device="cuda")
    room[:, :n] = l
    check_loss(experts.balance_loss(room[:, :n], plan), l, plan)


def test_balance_of_an_even_router_is_one():
    l = torch.zeros((256, 16), device="cuda")
    plan = experts.route(torch.eye(16, device="cuda").repeat(16, 1), 1)
    b = experts.balance_loss(l, plan)
    assert abs(float(b.loss) - 1.0) < 1e-6 and b.counts.tolist() == [16] * 16
    assert not experts.balance_loss_backward(torch.ones((), device="cuda"), l, b).abs().max() > 1e-9


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,n,k", SIZES)
def test_balance_loss_backward(tokens, n, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(7)
    l = logits_of(tokens + n, tokens, n, dtype)
    dloss = torch.full((), 3.0, device="cuda")
    dweights = torch.randn((tokens, k), generator=g, device="cuda") * 0.1
    p, there, d = softmax(l)
    for renormalize in (False, True):
        plan = experts.route(l, k, renormalize=renormalize)
        b = experts.balance_loss(l, plan)
        c = b.counts.double()
        scale = 3.0 * n / (max(1, int(c.sum())) * max(1, int(there.sum())))
        ex, r = (p * c).sum(1, keepdim=True), bound_of(p, d, n)
        er = (r * c).sum(1, keepdim=True) + (n / 32 + 6) * U * ex
        want = scale * p * (c - ex)
        bound = scale * (r * (c - ex).abs() + p * (er + 8 * U * (c + ex))) + 1e-37

        def within(got, exact, e):
            bad = ~((got.double() - exact).abs() <= e + HALF[dtype] * exact.abs() * 1.01 + TINY[dtype])
            assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}"
        within(experts.balance_loss_backward(dloss, l, b), want, bound)
        # with the router's gradient: the formula's, from the plan's weights
        ids, w = plan.experts.long(), plan.weights.double()
        ok = ids >= 0
        dw = torch.where(ok, dweights.double(), 0.0)
        mean, emean = (dw * w).sum(1, keepdim=True), 40 * U * (dw * w).abs().sum(1, keepdim=True)
        chosen = w * (dw - mean) if renormalize else w * dw
        both = want - (0 if renormalize else p * mean)
        both = both.scatter_add(1, ids.clamp(min=0), torch.where(ok, chosen, 0.0))
        e = bound + (0 if renormalize else r * mean.abs() + p * (emean + 4 * U * mean.abs())) + 4 * U * (want.abs() + p * mean.abs())
        e = e.scatter_add(1, ids.clamp(min=0), torch.where(ok, w * (emean + 6 * U * (dw.abs() + mean.abs())), 0.0))
        within(experts.balance_loss_backward(dloss, l, b, plan=plan, dweights=dweights), both, e)


def test_gradient_is_a_difference():
    """The kernels' gradient times a direction is the slope of the formula in 64 bits with the counts kept, as the definition has it."""
    l = logits_of(3, 40, 24, torch.float32, masked=False)
    plan = experts.route(l, 3)
    b = experts.balance_loss(l, plan)
    grad = experts.balance_loss_backward(torch.ones((), device="cuda"), l, b).double()
    c = b.counts.double()

    def loss(x):
        return float((torch.softmax(x, 1).mean(0) * c).sum()) * 24 / float(c.sum())
    direction = torch.randn(l.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.float64)
    slope = (loss(l.double() + 1e-5 * direction) - loss(l.double() - 1e-5 * direction)) / 2e-5
    size = float((grad.abs() * direction.abs()).sum())
    assert abs(slope - float((grad * direction).sum())) <= 1e-5 * size


def test_what_is_not_a_number_stays_in_its_row():
    l = logits_of(5, 100, 64, torch.float32)
    plan = experts.route(l, 4)
    b = experts.balance_loss(l, plan)
    want = experts.balance_loss_backward(torch.ones((), device="cuda"), l, b)
    bad = l.clone()
    bad[50, 3] = float("nan")
    got = experts.balance_loss_backward(torch.ones((), device="cuda"), bad, b)
    rest = torch.arange(100, device="cuda") != 50
    assert torch.equal(got[rest], want[rest]) and got[50].isnan().all()
    assert experts.balance_loss(bad, plan).loss.isnan()


def test_bound_and_captured():
    l = logits_of(6, 700, 64, torch.bfloat16)
    plan = experts.bind(experts.route, l, 2)
    loss = experts.bind(experts.balance_loss, l, plan.outputs)
    dl = torch.ones((), device="cuda")
    back = experts.bind(experts.balance_loss_backward, dl, l, loss.outputs)
    for c in (plan, loss, back):
        c.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.launch(), loss.launch(), back.launch()
    for seed in (1, 2):
        l.copy_(logits_of(seed, 700, 64, torch.bfloat16))
        graph.replay()
        p = experts.route(l, 2)
        b = experts.balance_loss(l, p)
        assert all(torch.equal(x, y) for x, y in zip(loss.outputs, b))
        assert torch.equal(back.outputs, experts.balance_loss_backward(dl, l, b))


def test_refusals():
    l = logits_of(1, 32, 16, torch.float32)
    plan = experts.route(l, 2)
    b, one, dw = experts.balance_loss(l, plan), torch.ones((), device="cuda"), torch.ones((32, 2), device="cuda")
    for call in (lambda: experts.balance_loss(l[:, :8], plan), lambda: experts.balance_loss(l[:8], plan), lambda: experts.balance_loss(l.double(), plan),
                 lambda: experts.balance_loss(l.t(), plan), lambda: experts.balance_loss(l.detach().requires_grad_(), plan),
                 lambda: experts.balance_loss_backward(torch.ones(1, device="cuda"), l, b), lambda: experts.balance_loss_backward(one, l[:, :8], b),
                 lambda: experts.balance_loss_backward(one, l, b, plan=plan), lambda: experts.balance_loss_backward(one, l, b, dweights=dw),
                 lambda: experts.balance_loss_backward(one, l, b, plan=plan, dweights=dw[:3]), lambda: experts.balance_loss_backward(one, l, b, out=l),
                 lambda: experts.balance_loss_backward(one.cpu(), l, b)):
        with pytest.raises(FlexSpmvError):
            call()
