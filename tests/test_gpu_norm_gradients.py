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
