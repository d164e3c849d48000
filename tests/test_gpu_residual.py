"""Layer norm with its residual sum and dropout, its gradients, and dropout (``flexspmv_b200.residual``) against plain implementations in 64 bits.

Bounds, u = 2^-24 the rounding of 32 bits.  A sum over a row is 16 values (of rows beyond 16384: width / 1024 + 8) in a thread, a tree of 5 and one of 5: an
error of DEPTH u of the sum of magnitudes.  What is elementwise has a few u.  One rounding to the result's type is added.  The bounds are put together in
the order in which the formulas are: see each test."""
import numpy as np
import pytest
import torch

from flexspmv_b200 import experts, residual
from flexspmv_b200.binding import FlexSpmvError
from tests.philox import keep_mask

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24, torch.float32: 1e-38}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def depth(width):
    return max(16, width // 1024 + 8) + 12


def normal(seed, shape, dtype, scale=1.0, offset=0.0):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale + offset).to(dtype)


def apart(t, gap):
    """The same values with rows further apart."""
    room = torch.full((t.shape[0], t.shape[1] + gap), float("nan"), dtype=t.dtype, device=t.device)
    room[:, : t.shape[1]] = t
    return room[:, : t.shape[1]]


def seed_of(a, b):
    return torch.tensor([a, b], dtype=torch.int64, device="cuda")


def keep_of(x, p, seed):
    return torch.from_numpy(keep_mask(x.shape[0], x.shape[1], p, *seed.tolist())).cuda()


def rounding(got, exact):
    return HALF[got.dtype] * exact.abs() * 1.01 + TINY[got.dtype]


def within(got, exact, bound):
    err = (got.double() - exact).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, the worst by {float((err / bound).max()):.3g} bounds"


def summed(x, r, p, seed):
    """The sum before the norm, and what it may be off by: a product, its factor and an addition."""
    s = x.double()
    if p > 0:
        s = torch.where(keep_of(x, p, seed), s / (1 - p), 0.0)
    es = 3 * U * s.abs()
    if r is not None:
        s = s + r.double()
        es = es + U * s.abs() * 1.01
    return s, es


def check_norm(out, x, w, b, eps, r, p, seed):
    s, es = summed(x, r, p, seed)
    n = x.shape[1]
    mean = s.mean(1, keepdim=True)
    c = s - mean
    var = (c * c).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    d = depth(n) * U
    em = d * s.abs().mean(1, keepdim=True) + es.mean(1, keepdim=True) + U * mean.abs()
    within(out.mean[:, None], mean, em + 1e-38)
    ec = em + es + U * (c.abs() + em)                                        # of a difference from the mean
    # the mean of squares: a sum's error, and twice the difference times its error
    rv = ((d + 3 * U) * (c.abs() + ec).pow(2).mean(1, keepdim=True) + 2 * (c.abs() * ec).mean(1, keepdim=True) + (ec * ec).mean(1, keepdim=True)) / (var + eps)
    assert float(rv.max()) < 0.5
    rr = rv * 0.75 + 4 * U                                                     # of the root's reciprocal: (1 + rv)^-1/2, within 0.75 rv for rv up to 0.5
    within(out.rstd[:, None], rstd, rr * rstd)
    scale = w.double().abs() if w is not None else 1.0
    y = c * rstd * (w.double() if w is not None else 1.0) + (b.double() if b is not None else 0.0)
    ey = scale * rstd * (ec * (1 + rr) + c.abs() * (rr + 2 * U)) + U * y.abs()
    within(out.y, y, ey + rounding(out.y, y))
    if r is None and p == 0:
        assert out.sum is None
    else:
        within(out.sum, s, es + rounding(out.sum, s))


SHAPES = [(1, 1), (1, 8), (3, 5), (7, 64), (9, 100), (65, 512), (5, 513), (33, 1000), (17, 1024), (12, 1025), (40, 2048), (3, 2051), (5, 4096), (4, 4099),
          (3, 8192), (2, 12001), (3, 16384), (2, 16392), (2, 20003), (400, 24), (3001, 40)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
def test_layer_norm(rows, width, dtype):
    x, r = normal(1, (rows, width), dtype, 1.5, 0.3), normal(2, (rows, width), dtype, 2.0, -0.5)
    seed = seed_of(-3 - width, (1 << 33) + rows)
    for param in {torch.float32, dtype}:
        w, b = normal(3, (width,), param, 0.2, 1.0), normal(4, (width,), param, 0.3)
        check_norm(residual.layer_norm(x, w, b, residual=r), x, w, b, 1e-5, r, 0.0, seed)
    check_norm(residual.layer_norm(x, eps=1e-3), x, None, None, 1e-3, None, 0.0, seed)
    check_norm(residual.layer_norm(x, w, None, residual=r, p=0.25, seed=seed), x, w, None, 1e-5, r, 0.25, seed)
    check_norm(residual.layer_norm(x, None, b, p=0.9, seed=seed), x, None, b, 1e-5, None, 0.9, seed)
    # rows apart and not on 16 bytes: the same bits, as sums go by columns alone where both take the same width of access
    for gap in (3, 8):
        a, c = residual.layer_norm(apart(x, gap), w, b, residual=apart(r, 2 * gap), p=0.25, seed=seed), (x, w, b, 1e-5, r, 0.25, seed)
        check_norm(a, *c)


# as many rows as are copied ahead, in every number of threads a row, on and off 16 bytes
MANY = [(10_003, 64), (9_700, 33), (10_001, 504), (5_001, 768), (5_003, 1001), (4_750, 1024), (2_501, 2048), (2_400, 2001), (1_301, 4096), (610, 8192), (330, 16384)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", MANY)
def test_layer_norm_of_many_rows(rows, width, dtype):
    x, r = normal(1, (rows, width), dtype, 1.5, 0.3), normal(2, (rows, width), dtype, 2.0, -0.5)
    w, b = normal(3, (width,), torch.float32, 0.2, 1.0), normal(4, (width,), torch.float32, 0.3)
    seed = seed_of(77, rows)
    for residual_rows, p in ((r, 0.2), (r, 0.0), (None, 0.0), (None, 0.5)):
        out = residual.layer_norm(x, w, b, residual=residual_rows, p=p, seed=seed)
        check_norm(out, x, w, b, 1e-5, residual_rows, p, seed)
        again = residual.layer_norm(x, w, b, residual=residual_rows, p=p, seed=seed)
        assert all(torch.equal(s, t) for s, t in zip(out, again) if s is not None)
    gap = 8 if width % 8 == 0 else 3
    check_norm(residual.layer_norm(apart(x, gap), None, None, residual=apart(r, gap), p=0.2, seed=seed), x, None, None, 1e-5, r, 0.2, seed)


def test_layer_norm_of_special_rows():
    x = normal(5, (8, 640), torch.bfloat16)
    x[0] = 0.0                                                               # no variance: 0 times 1 / sqrt(eps)
    x[1] = 3.0
    x[2, 7] = float("inf")
    x[3, 9] = float("nan")
    x[4] = 1e4
    x[4, ::2] = 1e4 + 64
    w, b = normal(6, (640,), torch.float32), normal(7, (640,), torch.float32)
    out = residual.layer_norm(x, w, b)
    assert torch.equal(out.y[0], b.bfloat16()) and torch.equal(out.y[1], b.bfloat16())
    assert not out.y[2].isfinite().any() and out.y[3].isnan().all()          # and no other row
    good = [0, 1, 4, 5, 6, 7]
    check_norm(residual.Normed(*[t[good] if t is not None else None for t in out]), x[good], w, b, 1e-5, None, 0.0, None)
    dropped = ~keep_of(x, 0.5, seed_of(1, 2))
    y = torch.where(dropped, float("nan"), x)                                # what is dropped is 0 whatever it was
    y[2:4] = torch.where(dropped[2:4], float("inf"), 1.0)
    assert residual.layer_norm(y, w, b, p=0.5, seed=seed_of(1, 2)).y.isfinite().all()
    assert torch.equal(residual.dropout(y, 0.5, seed_of(1, 2)) == 0, dropped | (y == 0))
    empty = residual.layer_norm(x[:0], w, b)
    assert empty.y.shape == (0, 640) and empty.mean.shape == (0,)


def check_backward(out, dy, x, w, mean, rstd, dsum, p, seed):
    n = x.shape[1]
    m, rs = mean.double()[:, None], rstd.double()[:, None]
    norm = (x.double() - m) * rs
    en = 3 * U * norm.abs()
    g = dy.double() * (w.double() if w is not None else 1.0)
    d = depth(n) * U
    m1, m2 = g.mean(1, keepdim=True), (g * norm).mean(1, keepdim=True)
    e1 = (d + 2 * U) * g.abs().mean(1, keepdim=True)
    e2 = (d + 7 * U) * (g * norm).abs().mean(1, keepdim=True)
    ds = rs * (g - m1 - norm * m2)
    eds = rs.abs() * (U * g.abs() + e1 + norm.abs() * e2 + 4 * U * (norm * m2).abs() + 4 * U * (g.abs() + m1.abs() + (norm * m2).abs()))
    if dsum is not None:
        ds = ds + dsum.double()
        eds = eds + U * ds.abs()
    within(out.dresidual, ds, eds + rounding(out.dresidual, ds))
    dx = ds if p == 0 else torch.where(keep_of(x, p, seed), ds / (1 - p), 0.0)
    within(out.dx, dx, (eds + 3 * U * ds.abs()) / (1 - p) + rounding(out.dx, dx))
    if w is None:
        assert out.dweight is None and out.dbias is None
        return
    # over rows: each 148th or more in a CTA's registers, then CTAs by 32 and a tree
    rd = (x.shape[0] // 148 + 1 + 8 + 740 // 32 + 1 + 5) * U
    dw, db = (dy.double() * norm).sum(0), dy.double().sum(0)
    within(out.dweight, dw, (rd + 4 * U) * (dy.double() * norm).abs().sum(0) + rounding(out.dweight, dw))
    within(out.dbias, db, rd * dy.double().abs().sum(0) + rounding(out.dbias, db))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES + [(5000, 40), (2000, 600), (700, 1500), (1000, 3001)])
def test_layer_norm_backward(rows, width, dtype):
    x, dy, dsum = normal(1, (rows, width), dtype, 1.5, 0.3), normal(2, (rows, width), dtype, 0.5, 0.1), normal(3, (rows, width), dtype)
    var, mean = torch.var_mean(x.double(), dim=1, correction=0)
    mean, rstd = mean.float(), ((var + 1e-5) ** -0.5).float()
    seed = seed_of(17, -1)
    for param in {torch.float32, dtype}:
        w = normal(4, (width,), param, 0.2, 1.0)
        check_backward(residual.layer_norm_backward(dy, x, w, mean, rstd), dy, x, w, mean, rstd, None, 0.0, None)
    out = residual.layer_norm_backward(dy, x, w, mean, rstd, dsum=dsum, p=0.3, seed=seed)
    check_backward(out, dy, x, w, mean, rstd, dsum, 0.3, seed)
    again = residual.layer_norm_backward(dy, x, w, mean, rstd, dsum=dsum, p=0.3, seed=seed)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    check_backward(residual.layer_norm_backward(apart(dy, 5), apart(x, 8), None, mean, rstd, dsum=apart(dsum, 1)), dy, x, None, mean, rstd, dsum, 0.0, None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", MANY)
def test_layer_norm_backward_of_many_rows(rows, width, dtype):
    x, dy, dsum = normal(1, (rows, width), dtype, 1.5, 0.3), normal(2, (rows, width), dtype, 0.5, 0.1), normal(3, (rows, width), dtype)
    var, mean = torch.var_mean(x.double(), dim=1, correction=0)
    mean, rstd = mean.float(), ((var + 1e-5) ** -0.5).float()
    w, seed = normal(4, (width,), torch.float32, 0.2, 1.0), seed_of(18, rows)
    for d, p in ((dsum, 0.2), (None, 0.0)):
        out = residual.layer_norm_backward(dy, x, w, mean, rstd, dsum=d, p=p, seed=seed)
        check_backward(out, dy, x, w, mean, rstd, d, p, seed)
        again = residual.layer_norm_backward(dy, x, w, mean, rstd, dsum=d, p=p, seed=seed)
        assert all(torch.equal(s, t) for s, t in zip(out, again))
    gap = 8 if width % 8 == 0 else 3
    out = residual.layer_norm_backward(apart(dy, gap), apart(x, 2 * gap), None, mean, rstd, dsum=apart(dsum, gap))
    check_backward(out, dy, x, None, mean, rstd, dsum, 0.0, None)


def test_layer_norm_gradients_are_differences():
    """Along a random direction, in the formula's 64 bits: the gradients that the kernels give, times the direction, are the slope of the forward formula."""
    rows, width, p, seed = 6, 96, 0.4, seed_of(5, 6)
    x, r, dy, dsum = (normal(s, (rows, width), torch.float32) for s in range(4))
    w, b = normal(5, (width,), torch.float32, 0.3, 1.0), normal(6, (width,), torch.float32)
    keep = keep_of(x, p, seed).double() / (1 - p)

    def loss(x, r, w, b):
        s = r + keep * x
        var, mean = torch.var_mean(s, dim=1, correction=0, keepdim=True)
        return float((((s - mean) * (var + 1e-5) ** -0.5 * w + b) * dy.double()).sum() + (s * dsum.double()).sum())

    n = residual.layer_norm(x, w, b, residual=r, p=p, seed=seed)
    g = residual.layer_norm_backward(dy, n.sum, w, n.mean, n.rstd, dsum=dsum, p=p, seed=seed)
    args, grads = [t.double() for t in (x, r, w, b)], (g.dx, g.dresidual, g.dweight, g.dbias)
    for i in range(4):
        direction = normal(20 + i, args[i].shape, torch.float64)
        step = 1e-5
        up, down = ([a + sign * step * direction if j == i else a for j, a in enumerate(args)] for sign in (1, -1))
        slope = (loss(*up) - loss(*down)) / (2 * step)
        # differences: the third derivative's step^2, some 1e-10 of the terms, and 64 bits over the step; gradients: 32-bit sums of some 100 values
        size = float((grads[i].double().abs() * direction.abs()).sum())
        assert abs(slope - float((grads[i].double() * direction).sum())) <= 200 * U * size + 1e-8 * size


def test_no_rows_have_no_gradient():
    x, w = torch.zeros((0, 96), device="cuda"), torch.ones(96, device="cuda")
    out = residual.layer_norm_backward(x, x, w, x[:, 0], x[:, 0])
    assert out.dx.shape == (0, 96) and not out.dweight.any() and not out.dbias.any()
    wide = torch.zeros((0, 20000), device="cuda")
    out = residual.layer_norm_backward(wide, wide, torch.ones(20000, device="cuda"), wide[:, 0], wide[:, 0])
    assert not out.dweight.any() and not out.dbias.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES + [(20000, 70), (1100, 4096)])
def test_dropout(rows, width, dtype):
    x, r = normal(8, (rows, width), dtype, 3.0), normal(9, (rows, width), dtype)
    seed = seed_of((1 << 62) + width, -(1 << 40) - rows)
    for p in (0.1, 0.5, 1 - 2.0 ** -10):
        for added in (None, r):
            s, es = summed(x, added, p, seed)
            if dtype == torch.float16:
                keep = s.abs() < 6e4                                         # a scaled value may leave the type
                within(residual.dropout(x, p, seed, residual=added)[keep], s[keep], (es + rounding(x, s))[keep])
            else:
                out = residual.dropout(x, p, seed, residual=added)
                within(out, s, es + rounding(out, s))
    # any strides give the same bits
    assert torch.equal(residual.dropout(apart(x, 1), 0.5, seed, residual=apart(r, 7)), residual.dropout(x, 0.5, seed, residual=r))
    assert torch.equal(residual.dropout(x, 0.0, seed), x)
    # and dropout inside the norm drops the same
    n = residual.layer_norm(x, residual=r, p=0.5, seed=seed)
    assert torch.equal(n.sum, residual.dropout(x, 0.5, seed, residual=r))


def test_dropout_of_many_values():
    """More than 2^32 pieces of work do not fit a device; a long matrix whose last values lie beyond 2^31 does."""
    rows, width = 270_001, 8192
    x = torch.ones((rows, width), dtype=torch.bfloat16, device="cuda")
    out = residual.dropout(x, 0.5, seed_of(3, 4))
    tail = keep_mask(rows, 8, 0.5, 3, 4)[-5:]
    assert np.array_equal((out[-5:, :8] != 0).cpu().numpy(), tail)
    assert abs(float((out[-1000:].float()).mean()) - 1.0) < 5 * (1.0 / (1000 * width)) ** 0.5


def test_replays_with_a_raised_offset_and_other_streams():
    x, r = normal(10, (64, 768), torch.bfloat16), normal(11, (64, 768), torch.bfloat16)
    w, b = normal(12, (768,), torch.float32), normal(13, (768,), torch.float32)
    seed = seed_of(9, 0)
    norm = experts.bind(residual.layer_norm, x, w, b, residual=r, p=0.2, seed=seed)
    n = norm.outputs
    back = experts.bind(residual.layer_norm_backward, x, n.sum, w, n.mean, n.rstd, dsum=r, p=0.2, seed=seed)
    drop = experts.bind(residual.dropout, x, 0.2, seed, residual=r)
    for c in (norm, back, drop):
        c.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm.launch(), back.launch(), drop.launch()
        seed[1] += 1
    want = []
    for i in range(3):
        s = seed_of(9, i)
        a = residual.layer_norm(x, w, b, residual=r, p=0.2, seed=s)
        want.append((*a, *residual.layer_norm_backward(x, a.sum, w, a.mean, a.rstd, dsum=r, p=0.2, seed=s), residual.dropout(x, 0.2, s, residual=r)))
    for i in range(3):
        graph.replay()
        for got, exact in zip((*norm.outputs, *back.outputs, drop.outputs), want[i]):
            assert torch.equal(got, exact)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x.mul_(2)
        doubled = residual.layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    check_norm(doubled, x, w, b, 1e-5, None, 0.0, None)


def test_refusals():
    x, w, seed = normal(1, (4, 64), torch.bfloat16), normal(2, (64,), torch.float32), seed_of(1, 2)
    s = residual.layer_norm(x, w, w)
    for call in (lambda: residual.layer_norm(x.double()), lambda: residual.layer_norm(x[0]), lambda: residual.layer_norm(x[:, :0]),
                 lambda: residual.layer_norm(x, w[:5]), lambda: residual.layer_norm(x, w.half()), lambda: residual.layer_norm(x, w, w.bfloat16()),
                 lambda: residual.layer_norm(x, w, w, eps=-1.0), lambda: residual.layer_norm(x, residual=x.float()),
                 lambda: residual.layer_norm(x, residual=x[:3]), lambda: residual.layer_norm(x, p=0.5), lambda: residual.layer_norm(x, p=1.0, seed=seed),
                 lambda: residual.layer_norm(x, p=0.5, seed=seed[:1]), lambda: residual.layer_norm(x, p=0.5, seed=seed.int()),
                 lambda: residual.layer_norm(x, p=0.5, seed=seed.cpu()), lambda: residual.layer_norm(x.t()), lambda: residual.layer_norm(x, w.cpu()),
                 lambda: residual.layer_norm(x.expand(4, 4, 64)[:, 0]), lambda: residual.layer_norm_backward(x, x[:3], w, s.mean, s.rstd),
                 lambda: residual.layer_norm_backward(x, x, w, s.mean[:3], s.rstd), lambda: residual.layer_norm_backward(x, x, w, s.mean, s.rstd.double()),
                 lambda: residual.layer_norm_backward(x, x, w, s.mean, s.rstd, dsum=x.float()), lambda: residual.dropout(x, 0.5, None),
                 lambda: residual.dropout(x, float("nan"), seed), lambda: residual.dropout(x, -0.1, seed), lambda: residual.dropout(x, 0.5, seed, out=x),
                 lambda: residual.dropout(x, 0.5, seed, out=torch.empty_like(x[:3])), lambda: residual.dropout(x, 0.5, seed, residual=x, out=x[:4]),
                 lambda: residual.layer_norm(x.detach().requires_grad_()), lambda: experts.bind(torch.add, x, x)):
        with pytest.raises(FlexSpmvError):
            call()
    with torch.no_grad():
        residual.layer_norm(x.detach().requires_grad_())
