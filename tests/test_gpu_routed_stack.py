"""The operators around a routed expert layer together, as a model runs them (``expert_layer.RoutedStack``, ``DecodingStack``).

Bounds.  In 32-bit rows the norm and dropout are compared as they are elsewhere; a stack of 16-bit matrices is compared with the same operations of torch in 64 bits on the
same choices of experts, by magnitudes: each 16-bit rounding is 2^-8 of a value, norms divide by the rows' deviations, which are about 1 here."""
import pytest
import torch
import torch.nn.functional as F

from flexspmv_b200 import adapters, experts, residual
from flexspmv_b200.expert_layer import (Adapter, DecodingStack, RoutedExperts, RoutedStack, Stacked, _stack_example, dropout, layer_norm, route_balanced,
                                        sum_norm, train_step)

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def test_functions_carry_the_operators_gradients():
    x, stream = normal(1, (50, 96)).requires_grad_(), normal(2, (50, 96)).requires_grad_()
    w, b = (normal(3, (96,), scale=0.2) + 1).requires_grad_(), normal(4, (96,)).requires_grad_()
    seed, dy, ds = torch.tensor([3, 4], device="cuda"), normal(5, (50, 96)), normal(6, (50, 96))
    total, y = sum_norm(x, stream, w, b, p=0.3, seed=seed)
    torch.autograd.backward([total, y], [ds, dy])
    with torch.no_grad():
        n = residual.layer_norm(x, w, b, residual=stream, p=0.3, seed=seed)
        g = residual.layer_norm_backward(dy, n.sum, w, n.mean, n.rstd, dsum=ds, p=0.3, seed=seed)
    assert torch.equal(total, n.sum) and torch.equal(y, n.y)
    for t, want in ((x, g.dx), (stream, g.dresidual), (w, g.dweight), (b, g.dbias)):
        assert torch.equal(t.grad, want)
        t.grad = None
    # against torch's own derivatives, with the dropout's mask as a factor
    keep = (residual.dropout(torch.ones_like(x), 0.3, seed) != 0).double() / 0.7
    args = [t.detach().double().requires_grad_() for t in (x, stream, w, b)]
    s = args[1] + keep * args[0]
    torch.autograd.backward([s, F.layer_norm(s, (96,), args[2], args[3])], [ds.double(), dy.double()])
    for got, t in zip((g.dx, g.dresidual, g.dweight, g.dbias), args):
        assert float((got.double() - t.grad).norm()) <= 100 * 2.0 ** -24 * float(t.grad.norm())
    layer_norm(x, w, b).backward(dy)
    args = [t.detach().double().requires_grad_() for t in (x, w, b)]
    F.layer_norm(args[0], (96,), args[1], args[2]).backward(dy.double())
    for t, want in zip((x, w, b), args):
        assert float((t.grad.double() - want.grad).norm()) <= 100 * 2.0 ** -24 * float(want.grad.norm())
        t.grad = None
    stream.grad = None
    dropout(x, 0.3, seed, stream).backward(dy)
    assert torch.equal(x.grad, residual.dropout(dy, 0.3, seed)) and torch.equal(stream.grad, dy)
    x.grad = None
    dropout(x, 0.3, seed).sum().backward()                                  # a gradient that is one value spread out
    assert torch.equal(x.grad, residual.dropout(torch.ones_like(dy), 0.3, seed))


def test_router_and_balance_share_one_gradient():
    logits = normal(7, (300, 24)).requires_grad_()
    dw = normal(8, (300, 3))
    plan, even = route_balanced(logits, 3, renormalize=True)
    ((plan.weights * dw).sum() + 5.0 * even.loss).backward()
    l = logits.detach().double().requires_grad_()
    p = torch.softmax(l, 1)
    ids = plan.experts.long()
    top = p.gather(1, ids)
    loss = 24 * (even.counts.double() * p.mean(0)).sum() / even.counts.sum()
    ((top / top.sum(1, keepdim=True) * dw).sum() + 5.0 * loss).backward()
    assert abs(float(even.loss.detach()) - float(loss.detach())) <= 1e-5
    assert float((logits.grad.double() - l.grad).norm()) <= 200 * 2.0 ** -24 * float(l.grad.norm())
    # the weights' gradient alone, the loss's alone
    for use in (lambda p, e: (p.weights * dw).sum(), lambda p, e: e.loss):
        logits.grad = None
        use(*route_balanced(logits, 3, renormalize=True)).backward()
        assert logits.grad.isfinite().all() and logits.grad.any()


def plain_stack(stack, x):
    d = lambda t: t.detach().double()
    s = x.double()
    n = F.layer_norm(s, s.shape[1:], d(stack.weight[0]), d(stack.bias[0]))
    loss = 0.0
    for i, layer in enumerate(stack.layers):
        logits = n @ d(layer.router).t()
        p = torch.softmax(logits, 1)
        routed = sum(p[:, e, None] * (F.silu(n @ d(layer.w1[e]).t()) @ d(layer.w2[e]).t()) for e in range(p.shape[1]))
        loss += float(p.mean(0).sum())                                       # every expert has every token
        s = s + routed + n @ d(stack.shared[i][0]).t()
        n = F.layer_norm(s, s.shape[1:], d(stack.weight[i + 1]), d(stack.bias[i + 1]))
    return n, loss


def test_stack_in_evaluation():
    stack = RoutedStack(128, 256, 8, 8, 2, generator=gen(9)).eval()          # every expert: no choice that a rounding could change
    x = normal(10, (70, 128), torch.bfloat16)
    with torch.no_grad():
        out = stack(x)
    want, loss = plain_stack(stack, x)
    # each layer: normed, hidden, its activation, results, their sum, the shared product, the sum and the stream are rounded: 8 roundings of values of about 1 to 3,
    # and what they change reaches the next layer through matrices of gain about 1: two layers, 2^-8 each, root of the sum of squares in the norm
    assert float((out.y.double() - want).norm() / want.norm()) <= 2 * 8 * 2.0 ** -8 / 2
    assert abs(float(out.loss) - loss) <= 2e-2 * loss
    experts.check()


def test_stack_trains_with_every_gradient():
    stack = RoutedStack(64, 128, 8, 2, 2, p=0.2, generator=gen(11))
    x, target = normal(12, (200, 64), torch.bfloat16), normal(13, (200, 64))
    mask = torch.ones(200, dtype=torch.bool, device="cuda")
    mask[5] = False
    out = stack(x, mask)
    assert isinstance(out, Stacked) and int(stack.seed[1]) == 2
    (F.mse_loss(out.y.float(), target) + 0.01 * out.loss).backward()
    for name, p in stack.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all() and p.grad.any(), name
        p.grad = None
    # what a masked token holds reaches nothing
    stack.seed[1] = 0
    bad = x.clone()
    bad[5] = float("nan")
    again = stack(bad, mask)
    assert torch.equal(again.y, out.y) and torch.equal(again.loss, out.loss)
    again.y.float().sum().backward()
    assert all(p.grad.isfinite().all() for p in stack.parameters())
    stack.zero_grad(set_to_none=True)
    # the same offsets drop the same places, others others
    stack.seed[1] = 0
    assert torch.equal(stack(x, mask).y, out.y) and not torch.equal(stack(x, mask).y, out.y)
    before = [p.detach().clone() for p in stack.parameters()]
    train_step(stack, x, target, learning_rate=0.1, max_norm=1.0)
    assert all(not torch.equal(a, b) for a, b in zip(before, stack.parameters()))
    experts.check()


def test_captured_training_step_drops_other_places_in_every_replay():
    stack = RoutedStack(64, 128, 8, 2, 2, p=0.3, generator=gen(18))
    x, target = normal(19, (160, 64), torch.bfloat16), normal(20, (160, 64))

    def step():
        out = stack(x)
        (F.mse_loss(out.y.float(), target) + 0.01 * out.loss).backward()

    want = []
    for offset in (2, 4):
        stack.seed[1] = offset
        step()
        want.append([p.grad.clone() for p in stack.parameters()])
        stack.zero_grad(set_to_none=True)
    stack.seed[1] = 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                               # two layers: the offset is 2 then
    torch.cuda.current_stream().wait_stream(side)
    stack.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for grads in want:
        for p in stack.parameters():
            p.grad.zero_()
        graph.replay()
        assert all(torch.equal(p.grad, g) for p, g in zip(stack.parameters(), grads))
    experts.check()


def test_decoding_stack_is_the_stack():
    stack = RoutedStack(256, 128, 16, 2, 2, generator=gen(14)).eval()
    for tokens in (1, 5):
        step = DecodingStack(stack, tokens)
        step.x.copy_(normal(tokens, (tokens, 256), torch.bfloat16))
        with torch.no_grad():
            want = stack(step.x.clone()).y
        assert torch.equal(step.launch(), want)
    experts.check()


def test_decoding_stack_with_adapters_in_a_graph():
    """Requests without an adapter as without any; a request's result does not depend on the others'; replays follow x and ids."""
    width, tokens, count, rank = 256, 6, 5, 16
    stack = RoutedStack(width, 128, 16, 2, 2, generator=gen(15)).eval()
    low = [Adapter(normal(20 + i, (count, rank, width), torch.bfloat16, 0.1), normal(30 + i, (count, width, rank), torch.bfloat16, 0.1),
                   torch.rand(count, generator=gen(40 + i), device="cuda")) for i in range(2)]
    step, bare = DecodingStack(stack, tokens, low), DecodingStack(stack, tokens)
    for s in (step, bare):
        s.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.launch()
    x = normal(16, (tokens, width), torch.bfloat16)
    for ids in ([-1] * 6, [0, 1, 2, 3, 4, -1], [4, -1, -1, 0, 0, 0]):
        step.x.copy_(x), bare.x.copy_(x)
        step.ids.copy_(torch.tensor(ids, dtype=torch.int32))
        graph.replay()
        got, want = step.y.clone(), bare.launch()
        for t, i in enumerate(ids):
            assert torch.equal(got[t], want[t]) == (i < 0)
        # the projection of the first layer against its operator
        n = residual.layer_norm(x, stack.weight[0].detach(), stack.bias[0].detach()).y
        plan = adapters.plan(step.ids, count)
        direct = adapters.project(n, stack.shared[0].detach()[0], low[0].a, low[0].b, plan, scale=low[0].scale)
        alone = [adapters.project(n[t:t + 1], stack.shared[0].detach()[0], low[0].a, low[0].b, adapters.plan(step.ids[t:t + 1], count), scale=low[0].scale)
                 for t in range(tokens)]
        assert torch.equal(direct, torch.cat(alone))
    experts.check()


def test_a_layer_without_balance_is_as_it_was():
    layer = RoutedExperts(64, 128, 8, 2, generator=gen(17))
    x = normal(18, (90, 64), torch.bfloat16)
    with torch.no_grad():
        y, even = layer(x, balance=True)
        assert torch.equal(layer(x), y) and int(even.counts.sum()) == 180


def test_example_runs():
    lines = list(_stack_example(steps=3, tokens=256, width=128, hidden=256, num_experts=8))
    assert lines[0].startswith("stack, step 2") and lines[-1].endswith("True")
