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
