"""The norms that carry gradients (``expert_layer.layer_norm``, ``sum_norm``), as a whole: forward and backward against torch's derivatives in 64 bits."""
import pytest
import torch
import torch.nn.functional as F

from flexspmv_b200 import residual
from flexspmv_b200.binding import FlexSpmvError
from flexspmv_b200.expert_layer import layer_norm, sum_norm

pytestmark = pytest.mark.gpu


def normal(seed, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("rows,width", [(1, 8), (50, 96), (300, 1001), (40, 2048), (3, 9000)])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("biased", [True, False])
def test_norms_without_weight_or_bias(weighted, biased, rows, width):
    """Every gradient that there is, and no other.  Sums of n values in 32 bits by parts are off by some n 2^-24 at the worst, a few 2^-24 as a norm."""
    x, stream = normal(1, (rows, width)).requires_grad_(), normal(2, (rows, width)).requires_grad_()
    w = (normal(3, (width,), scale=0.2) + 1).requires_grad_() if weighted else None
    b = normal(4, (width,)).requires_grad_() if biased else None
    dy, ds, seed = normal(5, (rows, width)), normal(6, (rows, width)), torch.tensor([3, 4], device="cuda")
    keep = (residual.dropout(torch.ones_like(dy), 0.3, seed) != 0).double() / 0.7
    for p in (None, 0.0, 0.3):
        leaves = [t for t in (x, stream if p is not None else None, w, b) if t is not None]
        doubles = {id(t): t.detach().double().requires_grad_() for t in leaves}
        d = lambda t: doubles[id(t)] if t is not None else None
        for t in leaves:
            t.grad = None
        if p is None:
            layer_norm(x, w, b).backward(dy)
            F.layer_norm(d(x), (width,), d(w), d(b)).backward(dy.double())
        else:
            torch.autograd.backward(sum_norm(x, stream, w, b, p=p, seed=seed if p else None), [ds, dy])
            s = d(stream) + (keep if p else 1.0) * d(x)
            torch.autograd.backward([s, F.layer_norm(s, (width,), d(w), d(b))], [ds.double(), dy.double()])
        for t in leaves:
            assert float((t.grad.double() - d(t).grad).norm()) <= 100 * 2.0 ** -24 * float(d(t).grad.norm())


def test_bias_alone_in_the_operator():
    dy, x = normal(7, (40, 136), torch.bfloat16), normal(8, (40, 136), torch.bfloat16)
    n = residual.layer_norm(x)
    for bias in (torch.zeros(136, device="cuda"), torch.zeros(136, dtype=torch.bfloat16, device="cuda")):
        g = residual.layer_norm_backward(dy, x, None, n.mean, n.rstd, bias=bias)
        assert g.dweight is None and g.dbias.dtype == bias.dtype
        with_ones = residual.layer_norm_backward(dy, x, torch.ones_like(bias), n.mean, n.rstd)
        assert torch.equal(g.dbias, with_ones.dbias) and torch.equal(g.dx, with_ones.dx)
    none = residual.layer_norm_backward(dy, x, None, n.mean, n.rstd)
    assert none.dweight is None and none.dbias is None and torch.equal(none.dx, g.dx)
    for bad in (torch.zeros(135, device="cuda"), torch.zeros(136, dtype=torch.float16, device="cuda")):
        with pytest.raises(FlexSpmvError, match="bias"):
            residual.layer_norm_backward(dy, x, None, n.mean, n.rstd, bias=bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("offset", [0.0, 10.0, 100.0])
@pytest.mark.parametrize("rows,width", [(40, 96), (300, 1001), (20, 4096)])
def test_sum_norm_as_a_whole(rows, width, offset, dtype):
    """Forward and backward in 16 bits against the derivative in 64 bits, rows whose mean is `offset` deviations among them.

    The backward pass has the sum as it was rounded, s + d with |d| <= h |s| (h half a step of the type) and the statistics of s: normed values n + m with
    m = d rstd.  With g = dy weight the gradient rstd (g - mean(g) - n mean(g n)) becomes one that is off by rstd (|n| mean(|g m|) + |m| |mean(g n)| +
    |m| mean(|g m|)), and dweight by the sum of |dy m|.  Its own roundings: half a step of the result, and of what a few sums in 32 bits lose (width / 32 + 40
    steps of 2^-24 of the magnitudes)."""
    half = torch.finfo(dtype).eps / 2
    x, stream = normal(11, (rows, width), dtype, 0.6), (normal(12, (rows, width), torch.float32, 0.8) + offset).to(dtype)
    w, b = normal(13, (width,), scale=0.2) + 1, normal(14, (width,))
    dy, ds, seed = normal(15, (rows, width), dtype), normal(16, (rows, width), dtype), torch.tensor([5, 6], device="cuda")
    keep = (residual.dropout(torch.ones_like(x), 0.25, seed) != 0).double() / 0.75
    leaves = [t.requires_grad_() for t in (x, stream, w, b)]
    torch.autograd.backward(sum_norm(x, stream, w, b, p=0.25, seed=seed), [ds, dy])
    doubles = [t.detach().double().requires_grad_() for t in leaves]
    s = doubles[1] + keep * doubles[0]
    torch.autograd.backward([s, F.layer_norm(s, (width,), doubles[2], doubles[3])], [ds.double(), dy.double()])
    s, g = s.detach(), dy.double() * w.detach().double()
    rstd = (s.var(1, correction=0, keepdim=True) + 1e-5) ** -0.5
    n, m = (s - s.mean(1, keepdim=True)) * rstd, half * s.abs() * rstd
    lost = (width / 32 + 40) * 2.0 ** -24
    mean = lambda t: t.mean(1, keepdim=True)
    # statistics: of a sum of magnitudes, through the deviation
    es = lost * (mean(s.abs()) + s.abs()) * rstd
    m = m + es
    off = rstd * (n.abs() * mean((g * m).abs()) + m * mean(g * n).abs() + m * mean((g * m).abs()))
    off = off + (lost + es.amax(1, keepdim=True)) * rstd * 4 * (g.abs() + mean(g.abs()) + n.abs() * mean((g * n).abs())) + 2.0 ** -22 * ds.double().abs()
    want = doubles[1].grad
    bound = off + half * 1.01 * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert ((stream.grad.double() - want).abs() <= bound).all()
    want = doubles[0].grad
    bound = off * keep + (half * 1.01 + 2.0 ** -22) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert ((x.grad.double() - want).abs() <= bound).all()
    sums = (rows / 32 + 40) * 2.0 ** -24
    bound = (dy.double() * m).abs().sum(0) + (2 * sums + es.amax()) * (dy.double() * n).abs().sum(0) + 2.0 ** -24 * doubles[2].grad.abs()
    assert ((w.grad.double() - doubles[2].grad).abs() <= bound).all()
    assert ((b.grad.double() - doubles[3].grad).abs() <= sums * dy.double().abs().sum(0)).all()
