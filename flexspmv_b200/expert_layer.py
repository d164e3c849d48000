"""A routed expert layer on the operators of ``experts``: training, and a decoding step on fixed buffers.

    y[t] = sum_j w[t, j] * W2[e] silu(W1[e] x[t]),   e = e[t, j] the j-th choice of a router,  w its renormalized softmax weights

``RoutedExperts`` is the module (differentiable once in x, the router's matrix, W1 and W2); ``train_step`` runs it forward and backward, clips all
gradients by their common norm and updates the weights; ``DecodingStep`` binds the layer to the buffers of a fixed number of tokens, whose
``launch()`` can be captured in a CUDA graph.  The reference has no counterpart: its models are stencils and finite volumes
(shallow_water_equation/swe_main.py:13-146).

    python -m flexspmv_b200.expert_layer        # a few training steps and a captured decoding step on synthetic data
"""
from __future__ import annotations

from typing import Iterable, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import experts


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


def route(logits: torch.Tensor, k: int, renormalize: bool = False) -> experts.Plan:
    """``experts.route`` whose weights carry a gradient to ``logits``."""
    return experts.Plan(*_Route.apply(logits, k, renormalize), renormalize)


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

    def forward(self, x: torch.Tensor, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``x`` (tokens, width).  ``mask`` (tokens) bool: tokens that are there; the others take no expert and give zeros."""
        rows = x.float()
        if mask is not None:                     # whatever lies there: a row's gradient of zeros times a NaN would be one in the router's
            rows = rows.masked_fill(~mask[:, None], 0.0)
        logits = rows @ self.router.t()
        if mask is not None:
            logits = logits.masked_fill(~mask[:, None], float("-inf"))
        plan = route(logits, self.k, renormalize=True)
        hidden = F.silu(grouped(x, self.w1, plan))
        return combine(grouped(hidden, self.w2, plan, gather=False), plan)


def train_step(layer: nn.Module, x: torch.Tensor, target: torch.Tensor, learning_rate: float, max_norm: float):
    """One step of gradient descent on the mean squared error: the loss and the gradients' norm before clipping, on the device."""
    loss = F.mse_loss(layer(x).float(), target.float())
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

    def __init__(self, layer: RoutedExperts, tokens: int):
        w1 = layer.w1.detach()
        self.x = torch.zeros((tokens, w1.shape[2]), dtype=w1.dtype, device=w1.device)
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


if __name__ == "__main__":
    for line in _example():
        print(line)
