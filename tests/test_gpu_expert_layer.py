"""The routed expert layer (``flexspmv_b200.expert_layer``) against the same layer in 64 bits with torch's own derivatives.

Bounds.  Every value that the layer keeps in 16 bits (hidden, its activation, the experts' results, their sum, and as many gradients) is one
rounding, 2^-8 of it, and reaches the result through matrices; with absolute values in the place of all factors the sum of their
effects is at most (number of roundings) * 2^-8 of the result's magnitude so computed.  silu and its derivative are below 1.1 |x| and 1.1,
its second derivative below 0.5: a rounding of the hidden values changes a gradient by at most half of its magnitude times theirs."""
import pytest
import torch
import torch.nn.functional as F

from flexspmv_b200 import experts
from flexspmv_b200.expert_layer import DecodingStep, RoutedExperts, _example, train_step

pytestmark = pytest.mark.gpu


def layer_of(seed, width, hidden, n, k):
    return RoutedExperts(width, hidden, n, k, generator=torch.Generator(device="cuda").manual_seed(seed))


def plain(x, router, w1, w2, k, mask):
    """The layer token by token of every expert, in the arguments' precision."""
    logits = x @ router.t()
    top = torch.topk(logits, k, dim=1)
    weights = torch.softmax(top.values, dim=1) * mask[:, None]
    out = torch.zeros_like(x)
    for e in range(w1.shape[0]):
        t, j = torch.nonzero(top.indices == e, as_tuple=True)
        out = out.index_add(0, t, weights[t, j, None] * (F.silu(x[t] @ w1[e].t()) @ w2[e].t()))
    return out


@pytest.mark.parametrize("tokens,width,hidden,n,k", [(1, 64, 128, 4, 2), (77, 128, 72, 8, 3), (600, 256, 512, 16, 2)])
def test_layer_and_its_gradients(tokens, width, hidden, n, k):
    layer = layer_of(1, width, hidden, n, k)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((tokens, width), generator=g, device="cuda").to(torch.bfloat16).requires_grad_()
    mask = torch.rand(tokens, generator=g, device="cuda") > (0.1 if tokens > 1 else -1.0)
    dy = torch.randn((tokens, width), generator=g, device="cuda").to(torch.bfloat16)
    y = layer(x, mask)
    y.backward(dy)
    experts.check()
    args = [t.detach().double().requires_grad_() for t in (x, layer.router, layer.w1, layer.w2)]
    want = plain(*args, k, mask.double())
    want.backward(dy.double())
    # magnitudes: the same sums of absolute values, silu(h) as 1.1 |h|
    ax, ar, a1, a2 = [t.detach().abs() for t in args]
    logits = args[0].detach() @ args[1].detach().t()
    top = torch.topk(logits, k, dim=1)
    w = torch.softmax(top.values, dim=1) * mask.double()[:, None]
    u = 2.0 ** -8
    my, mx = torch.zeros_like(ax), torch.zeros_like(ax)
    m1, m2 = torch.zeros_like(a1), torch.zeros_like(a2)
    reach = torch.zeros_like(w)                      # of dy through each choice's result
    ady = dy.double().abs()
    for e in range(n):
        t, j = torch.nonzero(top.indices == e, as_tuple=True)
        h, d = ax[t] @ a1[e].t(), w[t, j, None] * ady[t]
        z = 1.1 * h @ a2[e].t()
        my.index_add_(0, t, w[t, j, None] * z)
        dh = (1.1 + 0.5 * h) * (d @ a2[e])           # with the change of silu's derivative
        mx.index_add_(0, t, dh @ a1[e])
        m1[e], m2[e] = dh.t() @ ax[t], d.t() @ (1.1 * h)
        reach[t, j] = (ady[t] * z).sum(1)
    # the router's gradient: dw in full precision from rounded results, then a softmax
    dl = torch.zeros_like(logits).scatter_(1, top.indices, w * (reach + (w * reach).sum(1, keepdim=True)))
    assert bool(((y.double() - want).abs() <= 4 * u * my + 1e-30).all())
    assert bool(((x.grad.double() - args[0].grad).abs() <= 6 * u * (mx + dl @ ar) + 1e-30).all())
    assert bool(((layer.w1.grad.double() - args[2].grad).abs() <= 6 * u * m1 + 1e-30).all())
    assert bool(((layer.w2.grad.double() - args[3].grad).abs() <= 4 * u * m2 + 1e-30).all())
    assert bool(((layer.router.grad.double() - args[1].grad).abs() <= 4 * u * (dl.t() @ ax) + 1e-30).all())
    assert not y[~mask].any()


def test_train_step_clips_and_learns():
    layer = layer_of(3, 128, 256, 8, 2)
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((512, 128), generator=g, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        target = layer_of(5, 128, 256, 8, 2)(x)
    before = [p.detach().clone() for p in layer.parameters()]
    first, norm = train_step(layer, x, target, learning_rate=0.0, max_norm=1.0)
    assert all(torch.equal(a, p) for a, p in zip(before, layer.parameters())) and float(norm) > 0
    for _ in range(40):
        loss, _ = train_step(layer, x, target, learning_rate=5.0, max_norm=1.0)
    assert float(loss) < 0.8 * float(first)


def test_decoding_step_is_the_layer():
    layer = layer_of(6, 256, 128, 32, 4)
    for tokens in (1, 7):
        step = DecodingStep(layer, tokens)
        for seed in range(3):
            step.x.copy_(torch.randn(step.x.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))
            with torch.no_grad():
                want = layer(step.x.clone())
            assert torch.equal(step.launch(), want)
    experts.check()


def test_example_runs():
    lines = list(_example(steps=6, tokens=512, width=128, hidden=256, num_experts=8))
    assert lines[0].startswith("step 0") and lines[-1].endswith("True")
