"""Mean probabilities of experts whose logits are far below the largest, and the balance loss of tokens that lie on several devices.

Bounds, u = 2^-24: a power is off by 2^-22 and by d u for a logit d <= 8 below the largest, by 3 * 2 u beyond that; the sum that it is divided by by n / 32 + 5 additions
and as much as its largest powers; the mean by the tree of the tokens."""
import pytest
import torch

from flexspmv_b200 import experts

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("tokens,n", [(1, 8), (48, 64), (128, 60), (129, 256), (5000, 384), (700, 1024)])
def test_means_far_below_the_largest(tokens, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    below = torch.linspace(0.0, 85.0, n, device="cuda")                       # a step of an expert: the same for all tokens, but for a little
    l = 20.0 - below + torch.rand((tokens, n), generator=g, device="cuda") * 0.25
    b = experts.balance_loss(l, experts.route(l, 2))
    p = torch.softmax(l.double(), 1)
    want = p.mean(0)
    power = 4 * U + torch.clamp(below.double() + 0.25, max=8.0) * U
    power = torch.maximum(power, torch.full_like(power, 6 * U))
    tree = (tokens / 148 / 8 + 1 + 16 + 148 + 4) * U * (tokens > 128) + (tokens / 8 + 16) * U * (tokens <= 128)
    bound = (power + 12.3 * U + (n / 32 + 5) * U + 3 * U + tree) * want + 1e-44
    assert ((b.mean.double() - want).abs() <= bound).all(), float(((b.mean.double() - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_on_several_devices(dtype):
    """Each device has some of the tokens; the counts and tokens of all are added up before the backward pass: the gradient of the whole, within one more
    rounding of the scale, and with the router's on top."""
    g = torch.Generator(device="cuda").manual_seed(2)
    l = torch.randn((700, 40), generator=g, device="cuda").to(dtype)
    l[5] = l[650] = float("-inf")
    dw = torch.randn((700, 3), generator=g, device="cuda")
    dloss = torch.full((), 0.7, device="cuda")
    plan = experts.route(l, 3)
    whole = experts.balance_loss(l, plan)
    parts = [l[:300].contiguous(), l[300:].contiguous()]
    plans = [experts.route(p, 3) for p in parts]
    made = [experts.balance_loss(p, q) for p, q in zip(parts, plans)]
    counts, tokens = made[0].counts + made[1].counts, made[0].tokens + made[1].tokens
    assert torch.equal(counts, whole.counts) and torch.equal(tokens, whole.tokens) and int(tokens) == 698
    for with_router in (False, True):
        joined = []
        for p, q, b, d in zip(parts, plans, made, (dw[:300], dw[300:])):
            more = dict(plan=q, dweights=d.contiguous()) if with_router else {}
            joined.append(experts.balance_loss_backward(dloss, p, b._replace(counts=counts, tokens=tokens), **more))
        more = dict(plan=plan, dweights=dw) if with_router else {}
        assert torch.equal(torch.cat(joined), experts.balance_loss_backward(dloss, l, whole, **more))
    # the loss of all: of the counts and the sums of probabilities
    mean = sum(b.mean * b.tokens for b in made) / tokens
    loss = 40.0 / counts.sum() * (counts * mean).sum()
    assert abs(float(loss) - float(whole.loss)) <= 300 * U * float(loss)


def test_a_loss_may_be_added_to():
    """In place, as training steps do; and no result of the call keeps its workspace."""
    from flexspmv_b200.expert_layer import route_balanced
    logits = torch.randn((5000, 256), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").requires_grad_()
    plan, even = route_balanced(logits, 2)
    want, = torch.autograd.grad(3.0 * even.loss + plan.weights.sum(), logits)
    plan, even = route_balanced(logits, 2)
    loss = even.loss
    loss *= 3.0
    loss += plan.weights.sum()
    loss.backward()
    assert torch.equal(logits.grad, want)
    bound = experts.bind(experts.balance_loss, logits.detach(), plan._replace(weights=plan.weights.detach()))
    held = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in bound.outputs}
    assert sum(held.values()) == 4 * (2 + 2 * 256)
