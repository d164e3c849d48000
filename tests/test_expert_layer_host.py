"""The routed expert layer's derivatives without a GPU: the operators below them are replaced by plain ones on the CPU."""
import gc
import weakref

import pytest
import torch

from flexspmv_b200 import expert_layer, experts


def plain_route(logits, k, renormalize=False):
    """Like experts.route, all arrays of a plan are views of one buffer."""
    tokens, n = logits.shape
    top = torch.topk(logits.detach(), k, dim=1)
    weights = torch.softmax(top.values, dim=1) if renormalize else torch.gather(torch.softmax(logits.detach(), dim=1), 1, top.indices)
    buf = torch.empty(tokens * k, dtype=torch.int32)
    made = buf.view(torch.float32).view(tokens, k).copy_(weights)
    flat = top.indices.reshape(-1)
    order = torch.argsort(flat, stable=True)
    slots = torch.empty_like(flat)
    slots[order] = torch.arange(flat.numel())
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(flat, minlength=n).cumsum(0)])
    return experts.Plan(made, top.indices.int(), offsets.int(), (order // k).int(), slots.view(tokens, k).int(), renormalize)


def plain_route_backward(dweights, logits, plan, out=None):
    w, ids = plan.weights, plan.experts.long()
    mean = (w * dweights).sum(1, keepdim=True)
    if plan.renormalize:
        return torch.zeros_like(logits).scatter_(1, ids, w * (dweights - mean))
    return torch.softmax(logits, dim=1) * (torch.zeros_like(logits).scatter_(1, ids, dweights) - mean)


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(experts, "route", plain_route)
    monkeypatch.setattr(experts, "route_backward", plain_route_backward)


@pytest.mark.parametrize("renormalize", [False, True])
def test_a_plan_is_freed_with_its_last_use(plain, renormalize):
    """Nothing but the caller holds a plan after its backward pass: no cycle that only the collector would find."""
    logits = torch.randn((6, 5), generator=torch.Generator().manual_seed(1), requires_grad=True)
    gc.collect()
    gc.disable()
    try:
        for backward in (True, False):
            plan = expert_layer.route(logits, 2, renormalize=renormalize)
            alive = [weakref.ref(t) for t in plan[:5]]
            if backward:
                (plan.weights * torch.arange(12.0).view(6, 2)).sum().backward()
            del plan
            assert all(a() is None for a in alive)
    finally:
        gc.enable()


@pytest.mark.parametrize("renormalize", [False, True])
def test_route_gradient(plain, renormalize):
    logits = torch.randn((6, 5), generator=torch.Generator().manual_seed(2), requires_grad=True)
    g = torch.randn((6, 2), generator=torch.Generator().manual_seed(3))
    plan = expert_layer.route(logits, 2, renormalize=renormalize)
    (plan.weights * g).sum().backward()
    assert plan.renormalize == renormalize
    other = logits.detach().double().requires_grad_()
    p = torch.softmax(other, dim=1).gather(1, plan.experts.long())
    ((p / p.sum(1, keepdim=True) if renormalize else p) * g).sum().backward()
    assert torch.allclose(logits.grad.double(), other.grad, rtol=1e-5, atol=1e-6)


def plain_grouped(x, weight, offsets, rows=None, out=None):
    take = x if rows is None else x[rows.long()]
    return torch.cat([take[a:b] @ weight[e].t() for e, (a, b) in enumerate(zip(offsets[:-1].tolist(), offsets[1:].tolist()))])


def plain_dx(dy, weight, offsets, out=None):
    return plain_grouped(dy, weight.transpose(1, 2), offsets)


def plain_dw(dy, x, offsets, rows=None, dtype=None, out=None):
    take = x if rows is None else x[rows.long()]
    return torch.stack([dy[a:b].t() @ take[a:b] for a, b in zip(offsets[:-1].tolist(), offsets[1:].tolist())])


def plain_combine(z, slots, weights=None, out=None):
    picked = z[slots.long()]
    return (picked if weights is None else weights[..., None] * picked).sum(1)


def plain_combine_backward(dout, z, slots, weights, offsets):
    dz = torch.zeros_like(z)
    dz[slots.long().reshape(-1)] = (weights[..., None] * dout[:, None, :]).reshape(-1, z.shape[1])
    return dz, torch.einsum("th,tkh->tk", dout, z[slots.long()])


@pytest.fixture
def plain_layer(plain, monkeypatch):
    for name, f in (("grouped_matmul", plain_grouped), ("grouped_matmul_dx", plain_dx), ("grouped_matmul_dw", plain_dw), ("combine", plain_combine),
                    ("combine_backward", plain_combine_backward)):
        monkeypatch.setattr(experts, name, f)


def layer_inputs():
    g = torch.Generator().manual_seed(4)
    return [torch.randn(s, generator=g, requires_grad=True) for s in ((6, 8), (5, 8), (5, 16, 8))]


@pytest.mark.parametrize("part", ["route", "grouped", "combine"])
def test_second_derivatives_are_refused(plain_layer, part):
    """The backward passes are calls that autograd does not see into: derivatives of them are an error, not a wrong number."""
    x, router, w1 = layer_inputs()
    with torch.no_grad():
        fixed = plain_route(x @ router.t(), 2)
    if part == "route":
        first, made = router, expert_layer.route(x.detach() @ router.t(), 2).weights
    elif part == "grouped":
        first, made = w1, expert_layer.grouped(x.detach(), w1, fixed)
    else:
        z = torch.randn((12, 8), requires_grad=True)
        first, made = z, expert_layer.combine(z, fixed)
    # the result squared: the second derivative of a linear operator, too, is not zero
    (grad,) = torch.autograd.grad((made ** 2).sum(), first, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad((grad ** 2).sum(), first, retain_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (grad ** 2).sum().backward()


def test_first_derivatives(plain_layer):
    x, router, w1 = layer_inputs()
    plan = expert_layer.route(x @ router.t(), 2, renormalize=True)
    y = expert_layer.combine(expert_layer.grouped(x, w1, plan), plan)
    (y ** 2).sum().backward()
    others = [t.detach().clone().requires_grad_() for t in (x, router, w1)]
    logits = others[0] @ others[1].t()
    top = torch.topk(logits, 2, dim=1)
    want = torch.einsum("tk,tkn->tn", torch.softmax(top.values, dim=1), torch.einsum("tknc,tc->tkn", others[2][top.indices], others[0]))
    (want ** 2).sum().backward()
    assert torch.allclose(y, want, rtol=1e-4, atol=1e-5)
    for a, b in zip((x, router, w1), others):
        assert torch.allclose(a.grad, b.grad, rtol=1e-4, atol=1e-4)
