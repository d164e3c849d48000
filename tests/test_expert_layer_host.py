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
