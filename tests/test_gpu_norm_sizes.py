"""Norms of rows whose values are far from one, as large as 32 bits hold."""
import pytest
import torch

from flexspmv_b200 import residual

pytestmark = pytest.mark.gpu

WIDTHS = [1, 8, 33, 100, 264, 504, 520, 1000, 1001, 1032, 2001, 2056, 4000, 4104, 8200, 9001, 16392]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", WIDTHS)
def test_gradients_of_rows_whose_mean_is_many_deviations(width, dtype):
    """All values of a row alike and large: x - mean is 0, and the gradient rstd (g - mean(g)) + dsum.  The threads' columns beyond the width have x = 0, which is
    infinitely many deviations from the mean in 32 bits, and no part in it."""
    g = torch.Generator(device="cuda").manual_seed(width)
    for rows in (2, 700):
        x = torch.full((rows, width), 2.0 ** 127, device="cuda").to(dtype)
        dy, dsum = (torch.randn((rows, width), generator=g, device="cuda").to(dtype) for _ in range(2))
        w = torch.rand(width, generator=g, device="cuda") + 0.5
        mean, rstd = torch.full((rows,), 2.0 ** 127, device="cuda"), torch.full((rows,), 4.0, device="cuda")
        out = residual.layer_norm_backward(dy, x, w, mean, rstd, dsum=dsum)
        scaled = dy.double() * w.double()
        want = 4.0 * (scaled - scaled.mean(1, keepdim=True)) + dsum.double()
        # sums of `width` values and a few roundings in 32 bits, one to the type
        bound = 2.0 ** -24 * (width / 32 + 40) * (4.0 * (scaled.abs() + scaled.abs().mean(1, keepdim=True)) + dsum.abs().double()) + torch.finfo(dtype).eps / 2 * 1.01 * want.abs()
        assert ((out.dresidual.double() - want).abs() <= bound).all()
        assert not out.dweight.any()
        assert ((out.dbias.double() - dy.double().sum(0)).abs() <= rows * 2.0 ** -24 * dy.double().abs().sum(0)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [2.0 ** 62, 2.0 ** 66, 2.0 ** 100, 2.0 ** 123, 2.0 ** -40])
@pytest.mark.parametrize("width", WIDTHS)
def test_norms_of_rows_of_any_size(width, scale, dtype):
    """Rows whose squares, or whose sum, leave 32 bits, beside others; the norm of a scaled row is that of the row, for what eps counts.

    Bounds: a sum of `width` values of 32 bits, by parts, is off by (width / 32 + 40) 2^-24 of their magnitudes; the mean by that, a difference from it by as much,
    the root of the mean square by no more than the largest of the differences' errors; then y's rounding."""
    g = torch.Generator(device="cuda").manual_seed(width)
    for rows in (2, 700):
        x = torch.randn((rows, width), generator=g, device="cuda").add_(0.7).to(dtype)
        big = torch.arange(rows, device="cuda")[:, None] % 3 != 2
        x = torch.where(big, x.float() * scale, x.float()).to(dtype)
        r = torch.where(big, torch.randn((rows, width), generator=g, device="cuda") * scale, torch.ones((), device="cuda")).to(dtype)
        seed = torch.tensor([rows, width], device="cuda")
        for residual_rows, p in ((None, 0.0), (r, 0.0), (r, 0.5)):
            out = residual.layer_norm(x, residual=residual_rows, p=p, seed=seed)
            s = x.double()
            if p:
                s = torch.where(residual.dropout(torch.ones_like(x), p, seed) != 0, s / (1 - p), 0.0)
            if residual_rows is not None:
                s = s + residual_rows.double()
            mean = s.mean(1, keepdim=True)
            c = s - mean
            std = (c.pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
            e = (width / 32 + 40) * 2.0 ** -24 * s.abs().mean(1, keepdim=True) + 4 * 2.0 ** -24 * s.abs()
            off = (e.amax(1, keepdim=True) / std) + (width / 32 + 40) * 2.0 ** -24          # of the root, relative
            assert ((out.mean.double()[:, None] - mean).abs() <= e.amax(1, keepdim=True)).all()
            assert ((out.rstd.double()[:, None] * std - 1.0).abs() <= 2 * off + 2.0 ** -21).all()
            bound = (e + c.abs() * (2 * off + 2.0 ** -21)) / std + torch.finfo(dtype).eps / 2 * 1.01 * (c / std).abs() + 1e-38
            assert ((out.y.double() - c / std).abs() <= bound).all()
