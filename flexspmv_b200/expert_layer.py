"""A routed expert layer on the operators of ``experts``, and a stack of such layers on a residual stream: training, and a decoding step on fixed buffers.

    y[t] = sum_j w[t, j] * W2[e] silu(W1[e] x[t]),   e = e[t, j] the j-th choice of a router,  w its renormalized softmax weights

``RoutedExperts`` is the module (differentiable once in x, the router's matrix, W1 and W2); ``train_step`` runs it forward and backward, clips all
gradients by their common norm and updates the weights; ``DecodingStep`` binds the layer to the buffers of a fixed number of tokens, whose
``launch()`` can be captured in a CUDA graph.

``RoutedStack`` has a shared projection beside each layer of experts, and a dropout, the residual sum and a norm behind them, in one pass
(``residual.layer_norm``); its routers are balanced (``experts.balance_loss``).  ``DecodingStack`` is its step for requests that bring low-rank adapters for
the shared projections (``adapters.project``).  The reference has no counterpart: its models are stencils and finite volumes
(shallow_water_equation/swe_main.py:13-146).

    python -m flexspmv_b200.expert_layer        # a few training steps and a captured decoding step on synthetic data
"""
from __future__ import annotations

from typing import Iterable, NamedTuple, Optional, Sequence

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import adapters, experts, residual
from .binding import FlexSpmvError


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, renormalize):
        plan = experts.route(logits, k, renormalize=renormalize)
        # kept as autograd keeps outputs: on the context itself they, the node and the context would hold one another
        ctx.save_for_backward(logits, plan.weights, plan.experts, plan.offsets)
        ctx.renormalize = renormalize
        ctx.mark_non_differentiable(plan.experts, plan.offsets, plan.rows, plan.slots)
        return plan.weights, plan.experts, plan.offsets, plan.rows, plan.slots

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, *_):
        logits, weights, ids, offsets = ctx.saved_tensors
        plan = experts.Plan(weights, ids, offsets, None, None, ctx.renormalize)
        return experts.route_backward(dweights.contiguous(), logits, plan), None, None


class _RouteBalanced(torch.autograd.Function):
    """``_Route`` with the balance loss, whose gradients are one pass over the logits."""

    @staticmethod
    def forward(ctx, logits, k, renormalize):
        plan = experts.route(logits, k, renormalize=renormalize)
        balance = experts.balance_loss(logits, plan)
        ctx.save_for_backward(logits, plan.weights, plan.experts, plan.offsets, balance.counts, balance.tokens)
        ctx.renormalize = renormalize
        rest = (plan.experts, plan.offsets, plan.rows, plan.slots, balance.counts, balance.mean, balance.tokens)
        ctx.mark_non_differentiable(*rest)
        return (plan.weights, balance.loss, *rest)

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, dloss, *_):
        logits, weights, ids, offsets, counts, tokens = ctx.saved_tensors
        plan = experts.Plan(weights, ids, offsets, None, None, ctx.renormalize)
        balance = experts.Balance(None, counts, None, tokens)
        return experts.balance_loss_backward(dloss, logits, balance, plan=plan, dweights=dweights.contiguous()), None, None


class _Grouped(torch.autograd.Function):
    """``rows`` and ``slots`` of a plan: x's rows are tokens, and a token's gradients are added up; without them x's rows are places."""

    @staticmethod
    def forward(ctx, x, weight, offsets, rows, slots):
        ctx.save_for_backward(x, weight, offsets, rows, slots)
        return experts.grouped_matmul(x, weight, offsets, rows=rows)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, offsets, rows, slots = ctx.saved_tensors
        dy = dy.contiguous()
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = experts.grouped_matmul_dx(dy, weight, offsets)
            if rows is not None:
                dx = experts.combine(dx, slots)
        if ctx.needs_input_grad[1]:
            dw = experts.grouped_matmul_dw(dy, x, offsets, rows=rows, dtype=weight.dtype)
        return dx, dw, None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, slots, weights, offsets):
        ctx.save_for_backward(z, slots, weights, offsets)
        return experts.combine(z, slots, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        z, slots, weights, offsets = ctx.saved_tensors
        dz, dweights = experts.combine_backward(dout.contiguous(), z, slots, weights, offsets)
        return dz, None, dweights, None


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        out = residual.layer_norm(x, weight, bias, eps=eps)
        ctx.save_for_backward(x, weight, out.mean, out.rstd, bias if weight is None else None)
        ctx.has_bias = bias is not None
        return out.y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd, bias = ctx.saved_tensors
        g = residual.layer_norm_backward(dy.contiguous(), x, weight, mean, rstd, bias=bias)
        return g.dx, g.dweight, g.dbias if ctx.has_bias else None, None


class _SumNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, stream, weight, bias, eps, p, seed):
        out = residual.layer_norm(x, weight, bias, eps=eps, residual=stream, p=p, seed=seed)
        ctx.save_for_backward(out.sum, weight, out.mean, out.rstd, seed, bias if weight is None else None)
        ctx.p, ctx.has_bias = p, bias is not None
        return out.sum, out.y

    @staticmethod
    @once_differentiable
    def backward(ctx, dsum, dy):
        total, weight, mean, rstd, seed, bias = ctx.saved_tensors
        g = residual.layer_norm_backward(dy.contiguous(), total, weight, mean, rstd, dsum=dsum.contiguous(), p=ctx.p, seed=seed, bias=bias)
        return g.dx, g.dresidual, g.dweight, g.dbias if ctx.has_bias else None, None, None, None


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, stream):
        ctx.save_for_backward(seed)
        ctx.p = p
        return residual.dropout(x, p, seed, residual=stream)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        dx = residual.dropout(dout.contiguous(), ctx.p, *ctx.saved_tensors) if ctx.needs_input_grad[0] else None
        return dx, None, None, dout if ctx.needs_input_grad[3] else None


def route(logits: torch.Tensor, k: int, renormalize: bool = False) -> experts.Plan:
    """``experts.route`` whose weights carry a gradient to ``logits``."""
    return experts.Plan(*_Route.apply(logits, k, renormalize), renormalize)


def route_balanced(logits: torch.Tensor, k: int, renormalize: bool = False):
    """``experts.route`` and ``experts.balance_loss``: the plan, whose weights carry a gradient to ``logits``, and the balance, whose loss does."""
    weights, loss, ids, offsets, rows, slots, counts, mean, tokens = _RouteBalanced.apply(logits, k, renormalize)
    return experts.Plan(weights, ids, offsets, rows, slots, renormalize), experts.Balance(loss, counts, mean, tokens)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float = 1e-5) -> torch.Tensor:
    """``residual.layer_norm`` of ``x`` itself, with gradients for ``x`` and for ``weight`` and ``bias`` where they are given."""
    return _Norm.apply(x, weight, bias, eps)


def sum_norm(x: torch.Tensor, stream: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float = 1e-5, p: float = 0.0,
             seed: Optional[torch.Tensor] = None):
    """``stream + dropout(x)`` and its norm, with gradients.  ``seed`` must hold the same two values until the backward pass: give it a copy of one that is raised.

    The norm is of the sum as it is in 32 bits; what is kept of it for the backward pass is the sum that is returned, rounded to the rows' type.  In 16 bits the
    gradients are those of normalised values that are off by that rounding over the row's deviation: a 256th (bfloat16) of |s| / deviation at the most."""
    return _SumNorm.apply(x, stream, weight, bias, eps, p, seed)


def dropout(x: torch.Tensor, p: float, seed: torch.Tensor, stream: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual.dropout`` with gradients; ``seed`` as in ``sum_norm``."""
    return _Dropout.apply(x, p, seed, stream)


def grouped(x: torch.Tensor, weight: torch.Tensor, plan: experts.Plan, gather: bool = True) -> torch.Tensor:
    """``experts.grouped_matmul`` on a plan with gradients; ``gather``: x's rows are tokens, otherwise places."""
    return _Grouped.apply(x, weight, plan.offsets, plan.rows if gather else None, plan.slots if gather else None)


def combine(z: torch.Tensor, plan: experts.Plan) -> torch.Tensor:
    """``experts.combine`` on a plan with gradients for ``z`` and the plan's weights."""
    return _Combine.apply(z, plan.slots, plan.weights, plan.offsets)


class RoutedExperts(nn.Module):
    """``width`` and ``hidden``: multiples of 8.  The router's matrix and the logits are in 32 bits, the experts in ``dtype``."""

    def __init__(self, width: int, hidden: int, num_experts: int, k: int, dtype: torch.dtype = torch.bfloat16, device="cuda",
                 generator: Optional[torch.Generator] = None):
        super().__init__()
        self.k = k

        def matrix(*shape, dt):
            return nn.Parameter((torch.randn(shape, generator=generator, device=device) * shape[-1] ** -0.5).to(dt))

        self.router = matrix(num_experts, width, dt=torch.float32)
        self.w1 = matrix(num_experts, hidden, width, dt=dtype)
        self.w2 = matrix(num_experts, width, hidden, dt=dtype)

    def forward(self, x: torch.Tensor, mask: Optional[torch.Tensor] = None, balance: bool = False):
        """``x`` (tokens, width).  ``mask`` (tokens) bool: tokens that are there; the others take no expert and give zeros.  ``balance``: returns
        ``experts.Balance`` beside the result, over the tokens that are there."""
        rows = x.float()
        if mask is not None:                     # whatever lies there: a row's gradient of zeros times a NaN would be one in the router's
            rows = rows.masked_fill(~mask[:, None], 0.0)
        logits = rows @ self.router.t()
        if mask is not None:
            logits = logits.masked_fill(~mask[:, None], float("-inf"))
        if balance:
            plan, even = route_balanced(logits, self.k, renormalize=True)
        else:
            plan = route(logits, self.k, renormalize=True)
        hidden = F.silu(grouped(x, self.w1, plan))
        out = combine(grouped(hidden, self.w2, plan, gather=False), plan)
        return (out, even) if balance else out


class Stacked(NamedTuple):
    y: torch.Tensor              # the last norm
    loss: torch.Tensor           # () float32: the sum of the layers' balance losses


class RoutedStack(nn.Module):
    """``depth`` layers on a residual stream s, each reading the norm n of the stream and writing into it:

        s' = s + dropout(experts(n) + W n),   n' = norm(s')

    with a norm of its own in front of the first.  Norms and routers are in 32 bits, the matrices in ``dtype``.  Dropout is on in training mode; ``seed``
    (a seed and an offset, a buffer) is raised once a layer and step.  Stacks of one seed drop the same places: ranks that train together on tokens of their
    own take different ones.  A pass that is run again in the backward pass (``torch.utils.checkpoint``) would find the buffer raised and drop other places than
    its loss has, which is an error: give ``forward`` a seed then."""

    def __init__(self, width: int, hidden: int, num_experts: int, k: int, depth: int, p: float = 0.1, dtype: torch.dtype = torch.bfloat16, device="cuda",
                 generator: Optional[torch.Generator] = None, seed: int = 0):
        super().__init__()
        self.p = p
        self.layers = nn.ModuleList(RoutedExperts(width, hidden, num_experts, k, dtype=dtype, device=device, generator=generator) for _ in range(depth))
        self.shared = nn.ParameterList(
            nn.Parameter((torch.randn((1, width, width), generator=generator, device=device) * width ** -0.5).to(dtype)) for _ in range(depth))
        self.weight = nn.ParameterList(nn.Parameter(torch.ones(width, device=device)) for _ in range(depth + 1))
        self.bias = nn.ParameterList(nn.Parameter(torch.zeros(width, device=device)) for _ in range(depth + 1))
        self.register_buffer("seed", torch.tensor([seed, 0], dtype=torch.int64, device=device))

    def _next_seed(self) -> torch.Tensor:
        if torch._C._current_graph_task_id() != -1:          # the autograd engine runs this
            raise FlexSpmvError("a stack's forward pass is run again in a backward pass, with another offset than the first time: give forward a seed")
        used = self.seed.clone()
        self.seed[1] += 1
        return used

    def forward(self, x: torch.Tensor, mask: Optional[torch.Tensor] = None, seed: Optional[torch.Tensor] = None) -> Stacked:
        """``x`` (tokens, width) of the matrices' type.  ``mask`` (tokens) bool: tokens that are there; the others count as rows of zeros, whatever they hold.
        ``seed`` (two int64 values): takes the place of the stack's own, which is then neither read nor raised; layer i has its offset plus i."""
        if seed is not None:
            residual._vector(seed, "seed", (torch.int64,), 2, x.get_device(), "of seed and offset")
        if mask is not None:
            x = x.masked_fill(~mask[:, None], 0.0)
        all_tokens = torch.arange(2, dtype=torch.int32, device=x.device) * x.shape[0]          # made on the device: a step may be captured
        p = self.p if self.training else 0.0
        stream, normed, loss = x, layer_norm(x, self.weight[0], self.bias[0]), torch.zeros((), device=x.device)
        for i, layer in enumerate(self.layers):
            routed, even = layer(normed, mask, balance=True)
            z = routed + _Grouped.apply(normed, self.shared[i], all_tokens, None, None)
            used = None
            if p > 0.0:
                used = self._next_seed() if seed is None else torch.stack([seed[0], seed[1] + i])
            stream, normed = sum_norm(z, stream, self.weight[i + 1], self.bias[i + 1], p=p, seed=used)
            loss = loss + even.loss
        return Stacked(normed, loss)


def train_step(layer: nn.Module, x: torch.Tensor, target: torch.Tensor, learning_rate: float, max_norm: float, balance: float = 0.01):
    """One step of gradient descent on the mean squared error, for a stack with ``balance`` times its balance loss: the loss and the gradients' norm
    before clipping, on the device."""
    out = layer(x)
    if isinstance(out, Stacked):
        loss = F.mse_loss(out.y.float(), target.float()) + balance * out.loss
    else:
        loss = F.mse_loss(out.float(), target.float())
    loss.backward()
    params = [p for p in layer.parameters() if p.grad is not None]
    norm = experts.clip_grad_norm([p.grad for p in params], max_norm)
    with torch.no_grad():
        for p in params:
            p.add_(p.grad, alpha=-learning_rate)
            p.grad = None
    return loss.detach(), norm


class DecodingStep:
    """The layer on fixed buffers: write ``x`` (tokens, width), ``launch()``, read ``y``.  Nothing is allocated or checked per step."""

    def __init__(self, layer: RoutedExperts, tokens: int, x: Optional[torch.Tensor] = None):
        """``x``: the buffer to read, where something else writes it."""
        w1 = layer.w1.detach()
        if x is None:
            x = torch.zeros((tokens, w1.shape[2]), dtype=w1.dtype, device=w1.device)
        experts._tensor(x, "x", (w1.dtype,), 2, w1.get_device())
        if tuple(x.shape) != (tokens, w1.shape[2]):
            raise FlexSpmvError(f"x must have the shape {(tokens, w1.shape[2])}, not {tuple(x.shape)}")
        self.x = x
        self._router = layer.router.detach().t()          # a view: the bound step follows the weights
        self._x32 = torch.zeros(self.x.shape, dtype=torch.float32, device=w1.device)
        self._logits = torch.zeros((tokens, w1.shape[0]), dtype=torch.float32, device=w1.device)
        self._route = experts.bind(experts.route, self._logits, layer.k, renormalize=True)
        plan = self._route.outputs
        self._up = experts.bind(experts.grouped_matmul, self.x, w1, plan.offsets, rows=plan.rows)
        self._down = experts.bind(experts.grouped_matmul, self._up.outputs, layer.w2.detach(), plan.offsets)
        self._combine = experts.bind(experts.combine, self._down.outputs, plan.slots, plan.weights)
        self.y = self._combine.outputs

    def launch(self) -> torch.Tensor:
        self._x32.copy_(self.x)
        torch.mm(self._x32, self._router, out=self._logits)
        self._route.launch()
        F.silu(self._up.launch(), inplace=True)
        self._down.launch()
        return self._combine.launch()


class Adapter(NamedTuple):
    """Low-rank adapters of a shared projection, one for each request that names it."""
    a: torch.Tensor              # (adapters, rank, width)
    b: torch.Tensor              # (adapters, width, rank)
    scale: Optional[torch.Tensor] = None


class DecodingStack:
    """A ``RoutedStack`` on fixed buffers, each token with the adapters of its request: write ``x`` (tokens, width) and ``ids`` (tokens, -1: none), ``launch()``, read
    ``y``.  Without ``low_rank`` the projections are the stack's own.  Nothing is allocated or checked per step, nothing is dropped."""

    def __init__(self, stack: RoutedStack, tokens: int, low_rank: Optional[Sequence[Adapter]] = None):
        if low_rank and len(low_rank) != len(stack.layers):
            raise FlexSpmvError(f"adapters of {len(low_rank)} projections for {len(stack.layers)} layers")
        first = stack.shared[0].detach()
        width, device = first.shape[1], first.device
        self.x = torch.zeros((tokens, width), dtype=first.dtype, device=device)
        self.ids = torch.full((tokens,), -1, dtype=torch.int32, device=device)
        self._plan = experts.bind(adapters.plan, self.ids, low_rank[0].a.shape[0]) if low_rank else None
        all_tokens = torch.tensor([0, tokens], dtype=torch.int32, device=device)
        norm = experts.bind(residual.layer_norm, self.x, stack.weight[0].detach(), stack.bias[0].detach())
        self._first, self._layers = norm, []
        stream, normed = self.x, norm.outputs.y
        for i, layer in enumerate(stack.layers):
            routed = DecodingStep(layer, tokens, x=normed)
            matrix = stack.shared[i].detach()
            if low_rank:
                low = low_rank[i]
                shared = experts.bind(adapters.project, normed, matrix[0], low.a, low.b, self._plan.outputs, scale=low.scale)
            else:
                shared = experts.bind(experts.grouped_matmul, normed, matrix, all_tokens)
            norm = experts.bind(residual.layer_norm, shared.outputs, stack.weight[i + 1].detach(), stack.bias[i + 1].detach(), residual=stream)
            self._layers.append((routed, shared, norm))
            stream, normed = norm.outputs.sum, norm.outputs.y
        self.y = normed

    def launch(self) -> torch.Tensor:
        if self._plan is not None:
            self._plan.launch()
        self._first.launch()
        for routed, shared, norm in self._layers:
            z = routed.launch()
            shared.launch().add_(z)
            norm.launch()
        return self.y


def _example(steps: int = 20, tokens: int = 4096, width: int = 1024, hidden: int = 2048, num_experts: int = 16, k: int = 2) -> Iterable[str]:
    g = torch.Generator(device="cuda").manual_seed(0)
    layer, teacher = (RoutedExperts(width, hidden, num_experts, k, generator=g) for _ in range(2))
    x = torch.randn((tokens, width), generator=g, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        target = teacher(x)
    for i in range(steps):
        loss, norm = train_step(layer, x, target, learning_rate=30.0, max_norm=1.0)
        if i % 5 == 0 or i + 1 == steps:
            yield f"step {i}: loss {float(loss):.5f}, gradient norm {float(norm):.5f}"
    step = DecodingStep(layer, 8)
    step.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.launch()
    step.x.copy_(x[:8])
    graph.replay()
    with torch.no_grad():
        same = torch.allclose(step.y.float(), layer(x[:8]).float(), rtol=2.0 ** -6, atol=1e-3)
    experts.check()
    yield f"decoding step of 8 tokens from a CUDA graph agrees with the layer: {same}"


def _stack_example(steps: int = 10, tokens: int = 2048, width: int = 512, hidden: int = 1024, num_experts: int = 16, k: int = 2, depth: int = 2) -> Iterable[str]:
    g = torch.Generator(device="cuda").manual_seed(1)
    stack = RoutedStack(width, hidden, num_experts, k, depth, generator=g)
    x = torch.randn((tokens, width), generator=g, device="cuda").to(torch.bfloat16)
    target = torch.randn((tokens, width), generator=g, device="cuda")
    for i in range(steps):
        loss, norm = train_step(stack, x, target, learning_rate=0.1, max_norm=1.0)
    yield f"stack, step {steps - 1}: loss {float(loss):.5f}, gradient norm {float(norm):.5f}, balance {float(stack(x).loss.detach()) / depth:.3f}"
    stack.eval()
    low_rank = [Adapter(*(torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16) * 0.05 for shape in ((4, 16, width), (4, width, 16)))) for _ in range(depth)]
    step = DecodingStack(stack, 6, low_rank)
    step.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.launch()
    step.x.copy_(x[:6])
    step.ids.copy_(torch.tensor([-1, 0, 1, 2, 3, -1], dtype=torch.int32))
    graph.replay()
    with torch.no_grad():
        plain = stack(x[:6]).y
    same = [torch.allclose(step.y[i].float(), plain[i].float(), rtol=2.0 ** -5, atol=2.0 ** -5) for i in range(6)]
    experts.check()
    yield f"requests without adapters agree with the stack, those with them do not: {same == [True, False, False, False, False, True]}"


if __name__ == "__main__":
    for example in (_example, _stack_example):
        for line in example():
            print(line)
