"""The balance loss of a stack whose routers choose a few of their experts, over the tokens that are there."""
import pytest
import torch

from flexspmv_b200 import expert_layer, experts
from flexspmv_b200.expert_layer import RoutedStack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("masked", [False, True])
def test_loss_of_the_choices_that_were_made(masked, monkeypatch):
    """Against counts from each layer's own choices and probabilities in 64 bits from its own logits: 300 2^-24 of a loss (a sum over experts and tokens each).  Twice as
    many experts as are of use make the losses differ from one, which they would be of any router whose tokens choose all experts."""
    g = torch.Generator(device="cuda").manual_seed(21)
    stack = RoutedStack(64, 128, 12, 2, 3, p=0.2, generator=g)
    with torch.no_grad():
        for layer in stack.layers:
            layer.router[:6] += 0.15                       # with the norm's bias some experts are liked by all
        for b in stack.bias:
            b.add_(0.3)
    x = torch.randn((230, 64), generator=g, device="cuda").to(torch.bfloat16)
    mask = torch.rand(230, generator=g, device="cuda") < 0.7 if masked else None
    seen = []
    plain = expert_layer.route_balanced

    def watched(logits, k, renormalize=False):
        out = plain(logits, k, renormalize=renormalize)
        seen.append((logits.detach(), out[0].experts, out[1]))
        return out
    monkeypatch.setattr(expert_layer, "route_balanced", watched)
    loss = stack(x, mask).loss
    assert len(seen) == 3
    want = 0.0
    for logits, chosen, even in seen:
        there = torch.ones(230, dtype=torch.bool, device="cuda") if mask is None else mask
        assert (chosen[~there] == -1).all() and (chosen[there] >= 0).all()
        top = logits[there].double().topk(2, 1).indices
        assert torch.equal(top.sort(1).values, chosen[there].long().sort(1).values)
        counts = torch.bincount(chosen[there].long().reshape(-1), minlength=12).double()
        one = 12 / counts.sum() * (counts * torch.softmax(logits[there].double(), 1).mean(0)).sum()
        assert torch.equal(even.counts.double(), counts) and int(even.tokens) == int(there.sum())
        assert abs(float(even.loss.detach()) - float(one)) <= 300 * 2.0 ** -24 * float(one) and float(one) > 1.1
        want += float(one)
    assert abs(float(loss.detach()) - want) <= 300 * 2.0 ** -24 * want
    loss.backward()
    assert all(layer.router.grad.isfinite().all() and layer.router.grad.any() for layer in stack.layers)
    experts.check()
