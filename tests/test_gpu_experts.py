"""Operators of a routed expert layer (``flexspmv_b200.experts``) against plain implementations in 64 bits.

Bounds.  A sum of n products in 32 bits differs from the exact one by at most n * 2^-23 * (sum of the products' magnitudes): each of the n
additions rounds (or, in a matrix instruction, cuts) a partial sum that the sum of magnitudes bounds.  One rounding to 16 bits adds half
a unit: 2^-9 (bfloat16) or 2^-12 (float16) of the value, and 2^-25 below float16's normal range.  What is in whole numbers is equal."""
import math

import numpy as np
import pytest
import torch

from flexspmv_b200 import experts
from flexspmv_b200.binding import FlexSpmvError

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def close(got, exact, magnitude, terms):
    """Every value within the bound of the module's first lines."""
    bound = terms * 2.0 ** -23 * magnitude + HALF[got.dtype] * exact.abs() * 1.01 + (2.0 ** -25 if got.dtype == torch.float16 else 0.0) + 1e-30
    err = (got.double() - exact).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, the worst by {float((err / bound).max()):.3g} bounds"


def offsets_of(counts, start=0):
    return torch.tensor(np.concatenate([[start], start + np.cumsum(counts)]), dtype=torch.int32, device="cuda")


# ---- router ------------------------------------------------------------------------------------------------------

def plain_route(logits, k, renormalize):
    l = logits.double().cpu().numpy()
    tokens, n = l.shape
    ids = np.argsort(-l, axis=1, kind="stable")[:, :k] if tokens else np.zeros((0, k), dtype=np.int64)
    top = np.take_along_axis(l, ids, axis=1)
    ok = ~np.isneginf(top)
    base = np.where(np.isneginf(top[:, :1]), 0.0, top[:, :1])
    e = np.exp(l - base)
    chosen = np.where(ok, np.exp(top - base), 0.0)
    total = chosen.sum(1, keepdims=True) if renormalize else e.sum(1, keepdims=True)
    w = chosen / np.where(total == 0, 1, total)
    flat = np.where(ok, ids, -1).reshape(-1)
    pair = np.flatnonzero(flat >= 0)
    pair = pair[np.argsort(flat[pair], kind="stable")]
    rows, slots = np.full(flat.size, -1), np.full(flat.size, -1)
    rows[:pair.size] = pair // k
    slots[pair] = np.arange(pair.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[pair], minlength=n))])
    p = e / np.where(e.sum(1, keepdims=True) == 0, 1, e.sum(1, keepdims=True))
    return w, flat.reshape(tokens, k), offsets, rows, slots.reshape(tokens, k), p


ROUTES = [(0, 8, 2), (1, 1, 1), (1, 64, 8), (7, 60, 4), (64, 33, 6), (65, 8, 8), (333, 256, 8), (1000, 40, 1), (5001, 384, 7), (20011, 128, 2),
          (513, 1024, 32)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,n,k", ROUTES)
def test_route(tokens, n, k, dtype):
    for renormalize in (False, True):
        logits = normal(tokens + n, (tokens, n), dtype)                       # 16-bit logits tie often
        if tokens > 6:
            logits[2] = float("-inf")                                         # a row that may take no expert
            logits[3, 1:] = float("-inf")                                     # one expert only
            logits[4] = torch.finfo(dtype).min                                # masked by the lowest value: all alike
            logits[5, : n // 2] = 0.0
            logits[5, n // 2:] = -0.0                                         # equal, lowest index first
        plan = experts.route(logits, k, renormalize=renormalize)
        w, ids, offsets, rows, slots, _ = plain_route(logits, k, renormalize)
        assert np.array_equal(plan.experts.cpu().numpy(), ids)
        assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
        assert np.array_equal(plan.rows.cpu().numpy(), rows)
        assert np.array_equal(plan.slots.cpu().numpy(), slots)
        # n exponentials (2 units each) summed, one quotient: relative
        assert np.all(np.abs(plan.weights.double().cpu().numpy() - w) <= (n + 8) * 2.0 ** -23 * w + 1e-37)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [257, 300, 383, 384, 385, 500, 512, 516, 1000, 1023])
def test_route_of_many_experts(n, dtype):
    """Each number of keys a lane sorts, rows with and without wide loads; rising, falling and equal logits."""
    logits = normal(n, (301, n), dtype)
    logits[0] = torch.arange(n, device="cuda").to(dtype)
    logits[1] = -torch.arange(n, device="cuda").to(dtype)
    logits[2] = 1.0
    for k in (1, 9, 32):
        plan = experts.route(logits, k)
        w, ids, offsets, rows, slots, _ = plain_route(logits, k, False)
        assert np.array_equal(plan.experts.cpu().numpy(), ids) and np.array_equal(plan.slots.cpu().numpy(), slots)
        assert np.array_equal(plan.offsets.cpu().numpy(), offsets) and np.array_equal(plan.rows.cpu().numpy(), rows)
        assert np.all(np.abs(plan.weights.double().cpu().numpy() - w) <= (n + 8) * 2.0 ** -23 * w + 1e-37)


def test_route_of_a_part_of_a_wider_matrix_and_bound():
    wide = normal(3, (300, 96), torch.float32)
    logits = wide[:, 16:56]
    call = experts.bind(experts.route, logits, 5, renormalize=True)
    for _ in range(3):
        wide.copy_(torch.randn(wide.shape, generator=gen(int(wide[0, 0].abs() * 1e4)), device="cuda"))
        plan = call.launch()
        w, ids, offsets, rows, slots, _ = plain_route(logits, 5, True)
        assert np.array_equal(plan.experts.cpu().numpy(), ids) and np.array_equal(plan.slots.cpu().numpy(), slots)
        assert np.array_equal(plan.offsets.cpu().numpy(), offsets) and np.array_equal(plan.rows.cpu().numpy(), rows)


def test_route_of_nan_and_infinite_logits():
    logits = torch.zeros((3, 16), device="cuda")
    logits[0, 3], logits[1, 5] = float("nan"), float("inf")
    plan = experts.route(logits, 16)
    ids = plan.experts.cpu().numpy()
    assert 3 not in ids[0] and ids[0, -1] == -1 and ids[1, 0] == 5 and sorted(ids[2]) == list(range(16))
    assert torch.isnan(plan.weights[0, :15]).all() and torch.isnan(plan.weights[1, 0]) and not torch.isnan(plan.weights[2]).any()
    plan = experts.route(logits, 4, renormalize=True)
    assert torch.equal(plan.weights[0].cpu(), torch.full((4,), 0.25))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,n,k", ROUTES[1:])
def test_route_backward(tokens, n, k, dtype):
    for renormalize in (False, True):
        logits = normal(tokens + n, (tokens, n), dtype)
        if tokens > 6:
            logits[2] = float("-inf")
            logits[3, 1:] = float("-inf")
        g = normal(9, (tokens, k), torch.float32)
        plan = experts.route(logits, k, renormalize=renormalize)
        got = experts.route_backward(g, logits, plan)
        w, ids, _, _, _, p = plain_route(logits, k, renormalize)
        gd = np.where(ids >= 0, g.double().cpu().numpy(), 0.0)
        mean = (gd * w).sum(1, keepdims=True)
        d = np.zeros((tokens, n))
        t, j = np.nonzero(ids >= 0)
        if renormalize:
            d[t, ids[t, j]] = (w * (gd - mean))[t, j]
            scale = np.zeros((tokens, n))
            scale[t, ids[t, j]] = (w * (np.abs(gd) + (np.abs(gd) * w).sum(1, keepdims=True)))[t, j]
        else:
            d[t, ids[t, j]] = gd[t, j]
            scale = p * (np.abs(d) + (np.abs(gd) * w).sum(1, keepdims=True))
            d = p * (d - mean)
        close(got, torch.from_numpy(d).cuda(), torch.from_numpy(scale).cuda(), n + k + 24)


def test_route_backward_against_differences():
    logits = normal(1, (40, 24), torch.float32)
    logits[:, ::2] += 4.0                                   # the choice of 6 does not change under the step
    logits[:, :12:2] += 4.0
    g, d = normal(2, (40, 6), torch.float32), normal(3, (40, 24), torch.float32)
    for renormalize in (False, True):
        plan = experts.route(logits, 6, renormalize=renormalize)
        grad = experts.route_backward(g, logits, plan)
        h = 2.0 ** -6

        def f(step):
            # the weights of the same experts
            q = experts.route(logits + step * d, 6, renormalize=renormalize)
            full = torch.zeros_like(logits).scatter_(1, q.experts.long(), q.weights)
            return (g.double() * torch.gather(full, 1, plan.experts.long()).double()).sum(1)
        assert torch.equal(torch.sort(experts.route(logits + h * d, 6).experts)[0], torch.sort(plan.experts)[0])
        assert torch.equal(torch.sort(experts.route(logits - h * d, 6).experts)[0], torch.sort(plan.experts)[0])
        slope, want = (f(h) - f(-h)) / (2 * h), (grad * d).double().sum(1)
        # the third derivative of a softmax along d is below 6 max|d|^3 sum|g|; rounding of the weights over 2 h
        bound = g.abs().double().sum(1) * (h * h * d.abs().amax(1).double() ** 3 + 64 * 2.0 ** -23 / h)
        assert bool(((slope - want).abs() <= bound).all())


# ---- grouped products --------------------------------------------------------------------------------------------

GROUPS = [
    ([1], 8, 8), ([3], 128, 64), ([0, 0, 5, 0], 136, 72), ([1, 0, 127, 128, 129, 0, 300, 17, 256, 257], 264, 200),
    ([2, 1, 1, 3, 0, 1, 1, 1], 512, 1024), ([40, 700, 3], 1000, 416), ([16] * 33, 128, 136), ([1100], 256, 64), ([64, 31, 33, 32, 15, 16, 17, 8], 384, 2048),
    ([5] * 60, 2048, 128), ([300, 20, 0, 500] * 10, 1024, 192),          # many tiles for every CTA, narrow and wide
    ([3, 0, 9], 264, 4096), ([150, 90], 200, 2048), ([2000], 128, 264),          # few tiles and long sums
]


def grouped_case(counts, n, k, dtype, gather, seed=0, extra=0, start=0):
    """x, weight, offsets, rows, and of every place: its expert (-1: none) and its row of x."""
    slots = start + sum(counts) + extra
    tokens = max(1, slots // 2 + 3) if gather else slots
    x, w = normal(seed, (tokens, k), dtype), normal(seed + 1, (len(counts), n, k), dtype, k ** -0.5)
    rows = torch.randint(0, tokens, (slots,), generator=gen(seed + 2), device="cuda", dtype=torch.int32) if gather else None
    of = torch.full((slots,), -1, dtype=torch.int64)
    at = start
    for e, c in enumerate(counts):
        of[at:at + c] = e
        at += c
    take = rows.long() if gather else torch.arange(slots, device="cuda")
    return x, w, offsets_of(counts, start), rows, of, take


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,n,k", GROUPS)
def test_grouped_matmul(counts, n, k, dtype, gather):
    x, w, offsets, rows, of, take = grouped_case(counts, n, k, dtype, gather, extra=5, start=3)
    y = experts.grouped_matmul(x, w, offsets, rows=rows)
    experts.check()
    assert y.shape == (of.numel(), n) and y.dtype == dtype
    for e in range(-1, len(counts)):
        at = torch.nonzero(of == e).view(-1).cuda()
        if e < 0:
            assert not y[at].any()
            continue
        xe, we = x[take[at]].double(), w[e].double()
        close(y[at], xe @ we.t(), xe.abs() @ we.abs().t(), k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,n,k", GROUPS)
def test_grouped_matmul_dx(counts, n, k, dtype):
    _, w, offsets, _, of, _ = grouped_case(counts, n, k, dtype, False, extra=5, start=3)
    dy = normal(7, (of.numel(), n), dtype)
    dx = experts.grouped_matmul_dx(dy, w, offsets)
    experts.check()
    for e in range(-1, len(counts)):
        at = torch.nonzero(of == e).view(-1).cuda()
        if e < 0:
            assert not dx[at].any()
            continue
        d, we = dy[at].double(), w[e].double()
        close(dx[at], d @ we, d.abs() @ we.abs(), n)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("counts,n,k", GROUPS)
def test_grouped_matmul_dw(counts, n, k, dtype, out_dtype, gather):
    x, w, offsets, rows, of, take = grouped_case(counts, n, k, dtype, gather, extra=5, start=3)
    dy = normal(7, (of.numel(), n), dtype)
    dw = experts.grouped_matmul_dw(dy, x, offsets, rows=rows, dtype=out_dtype)
    experts.check()
    assert dw.shape == w.shape and dw.dtype == out_dtype
    for e in range(len(counts)):
        at = torch.nonzero(of == e).view(-1).cuda()
        d, xe = dy[at].double(), x[take[at]].double()
        close(dw[e], d.t() @ xe, d.abs().t() @ xe.abs(), max(1, counts[e]))


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("counts,n,k", [([3000, 0, 1, 4100, 257, 2000], 1560, 2624), ([1100] * 12, 2048, 4096), ([6000], 3400, 2560)])
def test_grouped_large(counts, n, k, gather):
    """Tiles of both accumulators, the last of them half a tile, a round by halves; sampled rows and matrices."""
    x, w, offsets, rows, of, take = grouped_case(counts, n, k, torch.bfloat16, gather, extra=3, start=1)
    dy = normal(7, (of.numel(), n), torch.bfloat16)
    y = experts.grouped_matmul(x, w, offsets, rows=rows)
    dw = experts.grouped_matmul_dw(dy, x, offsets, rows=rows)
    experts.check()
    assert not y[0].any() and not y[-3:].any()
    for e in range(len(counts)):
        at = torch.nonzero(of == e).view(-1).cuda()
        if counts[e] == 0:
            assert not dw[e].any()
            continue
        xe, we, d = x[take[at]].double(), w[e].double(), dy[at].double()
        close(y[at], xe @ we.t(), xe.abs() @ we.abs().t(), k)
        close(dw[e], d.t() @ xe, d.abs().t() @ xe.abs(), counts[e])


@pytest.mark.parametrize("counts,n,k", [([9001, 513, 512, 40], 264, 328), ([30_000], 128, 256)])
def test_grouped_matmul_dw_in_32_bits_over_many_rows(counts, n, k):
    """Parts of 512 rows, each by 32 matrix instructions that cut at most two units of their partial sum, then as many correctly rounded
    additions as there are parts: 64 * 2^-23 of the magnitude and 2^-24 for each part, whatever the number of rows."""
    x, _, offsets, _, of, _ = grouped_case(counts, n, k, torch.bfloat16, False)
    dy = normal(7, (of.numel(), n), torch.bfloat16)
    dw = experts.grouped_matmul_dw(dy, x, offsets, dtype=torch.float32)
    for e, c in enumerate(counts):
        at = torch.nonzero(of == e).view(-1).cuda()
        d, xe = dy[at].double(), x[at].double()
        want = d.t() @ xe
        close(dw[e], want, d.abs().t() @ xe.abs(), 64 + c / 1024)
        assert float((dw[e].double() - want).norm() / want.norm()) < 1.5e-6


@pytest.mark.parametrize("gather", [False, True])
def test_grouped_rows_of_others_do_not_leak(gather):
    """NaN and infinity in the rows of some experts, and of none, stay there: groups end inside tiles."""
    counts, n, k = [5, 61, 1, 200, 0, 130, 7], 256, 192
    x, w, offsets, rows, of, take = grouped_case(counts, n, k, torch.bfloat16, False, extra=9, start=2)
    if gather:
        rows = torch.randperm(of.numel(), generator=gen(5), device="cuda", dtype=torch.int32)
        take = rows.long()
    dy = normal(8, (of.numel(), n), torch.bfloat16)
    clean = (experts.grouped_matmul(x, w, offsets, rows=rows), experts.grouped_matmul_dx(dy, w, offsets),
             experts.grouped_matmul_dw(dy, x, offsets, rows=rows))
    x2, dy2, w2 = x.clone(), dy.clone(), w.clone()
    spoiled = (of == -1) | (of == 1) | (of == 5)
    at = torch.nonzero(spoiled).view(-1).cuda()
    x2[take[at]], dy2[at] = float("nan"), float("inf")
    w2[1], w2[5], w2[4] = float("nan"), float("inf"), float("nan")
    got = (experts.grouped_matmul(x2, w2, offsets, rows=rows), experts.grouped_matmul_dx(dy2, w2, offsets),
           experts.grouped_matmul_dw(dy2, x2, offsets, rows=rows))
    keep = torch.nonzero(~spoiled).view(-1).cuda()
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[1][keep], clean[1][keep])
    for e in (0, 2, 3, 4, 6):
        assert torch.equal(got[2][e], clean[2][e])
    none = torch.nonzero(of == -1).view(-1).cuda()
    assert not got[0][none].any() and not got[1][none].any()


def test_grouped_rows_apart():
    """Inputs that are column ranges of wider matrices."""
    counts, n, k = [30, 0, 170, 1], 136, 264
    x, w, offsets, rows, of, take = grouped_case(counts, n, k, torch.float16, True)
    dy = normal(4, (of.numel(), n), torch.float16)
    xs, ds = torch.full((x.shape[0], k + 40), float("nan"), dtype=x.dtype, device="cuda"), torch.full((dy.shape[0], n + 24), float("nan"), dtype=x.dtype, device="cuda")
    xs[:, 16:16 + k], ds[:, 8:8 + n] = x, dy
    xv, dv = xs[:, 16:16 + k], ds[:, 8:8 + n]
    assert torch.equal(experts.grouped_matmul(xv, w, offsets, rows=rows), experts.grouped_matmul(x, w, offsets, rows=rows))
    assert torch.equal(experts.grouped_matmul_dx(dv, w, offsets), experts.grouped_matmul_dx(dy, w, offsets))
    assert torch.equal(experts.grouped_matmul_dw(dv, xv, offsets, rows=rows), experts.grouped_matmul_dw(dy, x, offsets, rows=rows))


def test_grouped_gradients_against_differences():
    """Whole numbers so small that every product, sum and result is exact: the product is linear, so differences are its gradients."""
    counts, n, k = [3, 0, 40, 129], 64, 128
    small = lambda seed, shape: torch.randint(-1, 2, shape, generator=gen(seed), device="cuda").to(torch.bfloat16)
    _, _, offsets, rows, of, take = grouped_case(counts, n, k, torch.bfloat16, True)
    tokens = int(rows.max()) + 1
    x, w, dx, dwt, dy = small(1, (tokens, k)), small(2, (4, n, k)), small(3, (tokens, k)), small(4, (4, n, k)), small(5, (of.numel(), n))
    f = lambda a, b: (dy.double() * experts.grouped_matmul(a, b, offsets, rows=rows).double()).sum()
    gx = experts.grouped_matmul_dx(dy, w, offsets)
    assert float(f(x + dx, w) - f(x, w)) == float((gx.double() * dx[take].double()).sum())
    gw = experts.grouped_matmul_dw(dy, x, offsets, rows=rows)
    assert float(f(x, w + dwt) - f(x, w)) == float((gw.double() * dwt.double()).sum())


def test_grouped_results_are_the_same_every_time():
    counts, n, k = [1, 3, 0, 2, 1, 1, 700, 9], 512, 2048
    x, w, offsets, rows, of, _ = grouped_case(counts, n, k, torch.bfloat16, True)
    dy = normal(4, (of.numel(), n), torch.bfloat16)
    calls = (experts.bind(experts.grouped_matmul, x, w, offsets, rows=rows), experts.bind(experts.grouped_matmul_dx, dy, w, offsets),
             experts.bind(experts.grouped_matmul_dw, dy, x, offsets, rows=rows, dtype=torch.float32))
    first = [c.launch().clone() for c in calls]
    for _ in range(5):
        for c, want in zip(calls, first):
            c.outputs.fill_(float("nan"))
            assert torch.equal(c.launch(), want)


def test_grouped_on_two_streams_and_in_a_graph():
    counts, n, k = [1, 0, 2, 5, 1], 256, 512
    x, w, offsets, rows, of, _ = grouped_case(counts, n, k, torch.bfloat16, True)
    want = experts.grouped_matmul(x, w, offsets, rows=rows)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    calls = [experts.bind(experts.grouped_matmul, x, w, offsets, rows=rows) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                c.launch()
    torch.cuda.synchronize()
    assert all(torch.equal(c.outputs, want) for c in calls)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls[0].launch()
    for _ in range(3):
        x.mul_(2)                                             # a power of two: the result doubles exactly
        want = want * 2
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(calls[0].outputs, want)


def test_grouped_empty():
    w = normal(1, (4, 64, 32), torch.bfloat16)
    zero = torch.zeros(5, dtype=torch.int32, device="cuda")
    x, dy = torch.empty((0, 32), dtype=torch.bfloat16, device="cuda"), torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    assert experts.grouped_matmul(x, w, zero).shape == (0, 64) and experts.grouped_matmul_dx(dy, w, zero).shape == (0, 32)
    assert not experts.grouped_matmul_dw(dy, x, zero).any()
    x = normal(2, (6, 32), torch.bfloat16)
    assert not experts.grouped_matmul(x, w, zero).any()       # places, but no expert's
    experts.check()


def test_grouped_wrong_plans_are_noticed_on_the_device():
    counts, n, k = [4, 60, 9], 128, 1024
    x, w, offsets, rows, of, take = grouped_case(counts, n, k, torch.bfloat16, True)
    dy = normal(4, (of.numel(), n), torch.bfloat16)
    for wrong in ([0, 5, 3, 73], [0, 4, 64, 74], [-1, 4, 64, 73], [0, 2 ** 30, 64, 73], [0, 73, 0, 73]):
        for call in (lambda o: experts.grouped_matmul(x, w, o, rows=rows), lambda o: experts.grouped_matmul_dx(dy, w, o),
                     lambda o: experts.grouped_matmul_dw(dy, x, o, rows=rows)):
            call(torch.tensor(wrong, dtype=torch.int32, device="cuda"))
            with pytest.raises(FlexSpmvError, match="do not fit"):
                experts.check()
    for value in (-1, x.shape[0], 2 ** 31 - 1):
        bad = rows.clone()
        bad[70] = value
        for call in (lambda r: experts.grouped_matmul(x, w, offsets, rows=r), lambda r: experts.grouped_matmul_dw(dy, x, offsets, rows=r)):
            call(bad)
            with pytest.raises(FlexSpmvError, match="do not fit"):
                experts.check()
    experts.check()
    close(experts.grouped_matmul(x, w, offsets, rows=rows)[:4], x[take[:4]].double() @ w[0].double().t(), x[take[:4]].double().abs() @ w[0].double().abs().t(), k)


# ---- combine -----------------------------------------------------------------------------------------------------

def combine_case(tokens, k, width, dtype, seed=0, holes=True):
    pairs = tokens * k
    slots = torch.randperm(pairs, generator=gen(seed), device="cuda", dtype=torch.int32).view(tokens, k)
    used = pairs
    if holes and pairs > 4:
        used = pairs - pairs // 5                              # the last places are nobody's
        slots = torch.where(slots < used, slots, torch.full_like(slots, -1))
    return normal(seed + 1, (pairs, width), dtype), slots, torch.rand((tokens, k), generator=gen(seed + 2), device="cuda"), offsets_of([used // 2, 0, used - used // 2])


COMBINES = [(0, 2, 64), (1, 1, 8), (1, 8, 1), (3, 5, 7), (16, 8, 2048), (129, 4, 1000), (257, 3, 1001), (700, 32, 40), (2000, 2, 4096), (65, 9, 1032)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,k,width", COMBINES)
def test_combine(tokens, k, width, dtype):
    z, slots, weights, _ = combine_case(tokens, k, width, dtype)
    picked = torch.where((slots >= 0)[..., None], z[slots.clamp(min=0).long()].double(), 0.0) if tokens else torch.zeros((0, k, width), device="cuda").double()
    for w in (weights, None):
        wd = (w if w is not None else torch.ones_like(weights)).double()
        got = experts.combine(z, slots, w)
        assert got.shape == (tokens, width)
        close(got, torch.einsum("tk,tkh->th", wd, picked), torch.einsum("tk,tkh->th", wd, picked.abs()), k + 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,k,width", COMBINES[1:])
def test_combine_backward(tokens, k, width, dtype):
    z, slots, weights, offsets = combine_case(tokens, k, width, dtype)
    dout = normal(5, (tokens, width), dtype)
    on = slots >= 0
    for w in (weights, None):
        wd = (w if w is not None else torch.ones_like(weights)).double()
        dz, dw = experts.combine_backward(dout, z, slots, w, offsets)
        want = torch.zeros(z.shape, dtype=torch.float64, device="cuda")
        want[slots[on].long()] = (wd[..., None] * dout.double()[:, None, :])[on]
        close(dz, want, want.abs(), 1)
        picked = torch.where(on[..., None], z[slots.clamp(min=0).long()].double(), 0.0)
        close(dw, torch.einsum("th,tkh->tk", dout.double(), picked), torch.einsum("th,tkh->tk", dout.double().abs(), picked.abs()), width)


def test_combine_ignores_what_no_slot_names():
    z, slots, weights, offsets = combine_case(200, 4, 512, torch.bfloat16)
    dout = normal(5, (200, 512), torch.bfloat16)
    want, (dz, dw) = experts.combine(z, slots, weights), experts.combine_backward(dout, z, slots, weights, offsets)
    z[int(offsets[-1]):] = float("nan")
    weights[slots < 0] = float("nan")
    assert torch.equal(experts.combine(z, slots, weights), want)
    got = experts.combine_backward(dout, z, slots, weights, offsets)
    assert torch.equal(got[0], dz) and torch.equal(got[1], dw)
    beyond = slots.clone()
    beyond[0, 0] = 2 ** 31 - 1
    slots[0, 0] = -1
    assert torch.equal(experts.combine(z, beyond, weights), experts.combine(z, slots, weights))


def test_combine_rows_apart_and_differences():
    z, slots, weights, offsets = combine_case(50, 3, 64, torch.bfloat16, holes=False)
    z, d = torch.randint(-2, 3, z.shape, generator=gen(1), device="cuda").to(z.dtype), torch.randint(-2, 3, z.shape, generator=gen(2), device="cuda").to(z.dtype)
    weights = torch.randint(0, 4, slots.shape, generator=gen(3), device="cuda").float()
    dw = torch.randint(-1, 2, slots.shape, generator=gen(4), device="cuda").float()
    dout = torch.randint(-2, 3, (50, 64), generator=gen(5), device="cuda").to(z.dtype)
    wide, wide_out = torch.full((z.shape[0], 80), float("nan"), dtype=z.dtype, device="cuda"), torch.full((50, 72), float("nan"), dtype=z.dtype, device="cuda")
    wide[:, 8:72], wide_out[:, 3:67] = z, dout
    f = lambda a, b: (dout.double() * experts.combine(a, slots, b).double()).sum()
    gz, gw = experts.combine_backward(wide_out[:, 3:67], wide[:, 8:72], slots, weights, offsets)
    assert torch.equal(experts.combine(wide[:, 8:72], slots, weights), experts.combine(z, slots, weights))
    assert float(f(z + d, weights) - f(z, weights)) == float((gz.double() * d.double()).sum())
    assert float(f(z, weights + dw) - f(z, weights)) == float((gw.double() * dw.double()).sum())


# ---- norm and clipping -------------------------------------------------------------------------------------------

def tensors_of(sizes, dtypes, seed=0, scale=1e-2):
    return [normal(seed + i, (s,), dtypes[i % len(dtypes)], scale) for i, s in enumerate(sizes)]


CLIPS = [[1], [0, 5], [4095, 4096, 4097], [3, 1_000_003, 17], list(range(1, 120)), [100_000, 7] * 160, [33] * 1000, [50] * 1001 + [8192] * 20, [40_000_019]]


@pytest.mark.parametrize("case", range(len(CLIPS)))
def test_norm_and_clip(case):
    sizes = CLIPS[case]
    mixed = [torch.float32, torch.bfloat16, torch.float16]
    ts = tensors_of(sizes, mixed, seed=case * 2000)
    exact = math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in ts))
    # a thread adds at most 65536 / 256 squares in 32 bits, then 64 bits are used: 2^-24 of 256 each, and a square root
    tol = 300 * 2.0 ** -24
    norm = experts.grad_norm(ts)
    assert norm.dtype == torch.float32 and abs(float(norm) - exact) <= tol * exact
    assert torch.equal(experts.grad_norm(ts), norm)
    for max_norm in (exact / 3, exact * 2):
        scale = min(1.0, max_norm / (exact + 1e-6))
        outs = [torch.full_like(t, float("nan"), dtype=mixed[(i // 3) % 3]) for i, t in enumerate(ts)]
        mine = [t.clone() for t in ts]
        assert torch.equal(experts.clip_grad_norm(ts, max_norm, out=outs), norm) and torch.equal(experts.clip_grad_norm(mine, max_norm), norm)
        for t, o, m in zip(ts, outs, mine):
            for got in (o, m):
                want = t.double() * scale
                low = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
                assert bool(((got.double() - want).abs() <= (HALF[got.dtype] * 1.01 + tol + 2.0 ** -22) * want.abs() + low).all())
        if scale == 1.0:
            assert all(torch.equal(a, b) for a, b in zip(mine, ts))


def test_clip_of_tensors_off_the_16_byte_grid():
    base = [normal(i, (5000 + i,), dt, 0.1) for i, dt in enumerate([torch.float32, torch.bfloat16, torch.float16, torch.bfloat16])]
    views, copies = [b[1 + i:] for i, b in enumerate(base)], [b[1 + i:].clone() for i, b in enumerate(base)]
    first = [b[:1].clone() for b in base]
    n1, n2 = experts.clip_grad_norm(views, 0.5), experts.clip_grad_norm(copies, 0.5)
    assert abs(float(n1) - float(n2)) <= 1e-5 * float(n2)
    assert all(torch.allclose(v.float(), c.float(), rtol=2.0 ** -7, atol=0) for v, c in zip(views, copies))
    assert all(torch.equal(b[:1], f) for b, f in zip(base, first))


def test_clip_of_infinite_and_nan_gradients():
    t = [torch.ones(5000, device="cuda"), torch.ones(3, device="cuda")]
    t[0][7] = float("inf")
    assert float(experts.clip_grad_norm(t, 1.0)) == float("inf")
    assert torch.isnan(t[0][7]) and float(t[0][0]) == 0.0 and float(t[1][1]) == 0.0
    t = [torch.ones(5000, device="cuda"), torch.ones(3, device="cuda")]
    t[1][2] = float("nan")
    assert math.isnan(float(experts.clip_grad_norm(t, 1.0))) and torch.isnan(t[0]).all()
    big = [torch.full((4096,), 1e18, device="cuda"), torch.full((1 << 22,), 1e17, device="cuda")]
    exact = math.sqrt(4096 * 1e36 + (1 << 22) * 1e34)
    assert abs(float(experts.grad_norm(big)) - exact) <= 1e-5 * exact


def test_bound_clip_follows_its_tensors():
    ts = tensors_of([1000, 3, 70_000], [torch.bfloat16])
    outs = [torch.empty(t.shape, device="cuda") for t in ts]
    call = experts.bind(experts.clip_grad_norm, ts, 1.0, out=outs)
    for i in range(3):
        for t in ts:
            t.mul_(2)
        norm = float(call.launch())
        exact = math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))
        assert abs(norm - exact) <= 1e-4 * exact
        assert all(torch.allclose(o, t.float() * min(1.0, 1.0 / (exact + 1e-6)), rtol=1e-4) for o, t in zip(outs, ts))


def test_bound_calls_on_another_stream():
    """Bound on one stream and launched on another at once: the plan comes first."""
    ts = tensors_of([300_000, 17], [torch.bfloat16])
    exact = math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        torch.cuda._sleep(1_000_000)                            # the binding stream is busy before the plan
        call = experts.bind(experts.grad_norm, ts)
        with torch.cuda.stream(side):
            norm = call.launch().clone()
        side.synchronize()
        assert abs(float(norm) - exact) <= 1e-4 * exact
        torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    call = experts.bind(experts.grad_norm, ts)
    with pytest.raises(FlexSpmvError, match="captured"):
        with torch.cuda.graph(graph):
            call.launch()


# ---- beyond 32 bits ----------------------------------------------------------------------------------------------

def test_arrays_of_more_than_2_to_the_32_values():
    """600 000 rows of 8192: the last group's rows lie beyond 2^32 values, in every operand that can be so long."""
    counts, n, k = [1000, 598_800, 200], 8192, 64
    slots = sum(counts)
    x, w = normal(1, (slots, k), torch.bfloat16), normal(2, (3, n, k), torch.bfloat16, 0.125)
    offsets = offsets_of(counts)
    y = experts.grouped_matmul(x, w, offsets)
    last = slice(slots - 200, slots)
    xe, we = x[last].double(), w[2].double()
    close(y[last], xe @ we.t(), xe.abs() @ we.abs().t(), k)
    xm = x[550_000:550_100].double()
    close(y[550_000:550_100], xm @ w[1].double().t(), xm.abs() @ w[1].double().abs().t(), k)
    dx = experts.grouped_matmul_dx(y, w, offsets)
    d = y[last].double()
    close(dx[last], d @ we, d.abs() @ we.abs(), n)
    dw = experts.grouped_matmul_dw(y, x, offsets, dtype=torch.float32)
    close(dw[2], d.t() @ xe, d.abs().t() @ xe.abs(), 200)
    rows = torch.arange(slots - 200, slots, device="cuda", dtype=torch.int32)          # taken from the far end of a long x
    dw = experts.grouped_matmul_dw(xe.to(torch.bfloat16), y, offsets_of([200]), rows=rows, dtype=torch.float32)
    close(dw[0], xe.t() @ d, xe.abs().t() @ d.abs(), 200)
    w2 = normal(3, (1, 64, n), torch.bfloat16, n ** -0.5)
    close(experts.grouped_matmul(y, w2, offsets_of([200]), rows=rows), d @ w2[0].double().t(), d.abs() @ w2[0].double().abs().t(), n)
    slots2 = torch.arange(slots, device="cuda", dtype=torch.int32).view(-1, 2)
    weights = torch.rand(slots2.shape, generator=gen(4), device="cuda")
    out = experts.combine(y, slots2, weights)
    picked = y[last].double().view(100, 2, n)
    close(out[-100:], torch.einsum("tk,tkh->th", weights[-100:].double(), picked), torch.einsum("tk,tkh->th", weights[-100:].double(), picked.abs()), 3)
    dz, dweights = experts.combine_backward(out, y, slots2, weights, offsets)
    want = (weights[-100:].double()[..., None] * out[-100:].double()[:, None, :]).reshape(200, n)
    close(dz[last], want, want.abs(), 1)
    close(dweights[-100:], torch.einsum("th,tkh->tk", out[-100:].double(), picked), torch.einsum("th,tkh->tk", out[-100:].double().abs(), picked.abs()), n)
    experts.check()
    long = y.view(-1)[: (1 << 32) + 12_345]
    long.fill_(0.5)
    norm = experts.clip_grad_norm([long], 1.0)
    assert abs(float(norm) - 0.5 * math.sqrt(long.numel())) <= 1e-5 * float(norm)
    scaled = (torch.tensor(0.5) * (1.0 / (norm.cpu() + 1e-6))).to(torch.bfloat16)
    assert float(long[-1]) == float(scaled) and float(long[0]) == float(scaled) and float(y.view(-1)[long.numel()]) != float(scaled)


# ---- refusals ----------------------------------------------------------------------------------------------------

def test_refusals():
    bf = torch.bfloat16
    x, w, off = normal(1, (10, 64), bf), normal(2, (3, 32, 64), bf), offsets_of([2, 3, 5])
    rows = torch.zeros(10, dtype=torch.int32, device="cuda")
    dy, logits = normal(3, (10, 32), bf), normal(4, (10, 16), torch.float32)
    plan = experts.route(logits, 2)
    z, slots = normal(5, (20, 64), bf), plan.slots
    for bad in (
        lambda: experts.route(logits.cpu(), 2), lambda: experts.route(logits.double(), 2), lambda: experts.route(logits, 0),
        lambda: experts.route(logits, 17), lambda: experts.route(logits.t(), 2), lambda: experts.route(logits[0], 1),
        lambda: experts.route(torch.zeros((2, 1025), device="cuda"), 2), lambda: experts.route(torch.zeros((2, 64), device="cuda"), 33),
        lambda: experts.route_backward(plan.weights[:5], logits, plan), lambda: experts.route_backward(plan.weights.half(), logits, plan),
        lambda: experts.grouped_matmul(x.float(), w.float(), off), lambda: experts.grouped_matmul(x, w.half(), off),
        lambda: experts.grouped_matmul(x[:, :56], w, off), lambda: experts.grouped_matmul(x, w, off[:3]), lambda: experts.grouped_matmul(x, w, off.long()),
        lambda: experts.grouped_matmul(x, w, off, rows=rows.long()), lambda: experts.grouped_matmul(x, w, off.cpu()),
        lambda: experts.grouped_matmul(x, w.transpose(1, 2), off), lambda: experts.grouped_matmul(x[:, :60], w[:, :, :60].contiguous(), off),
        lambda: experts.grouped_matmul(x.t().contiguous().t(), w, off), lambda: experts.grouped_matmul(x, w, off, out=dy[:5]),
        lambda: experts.grouped_matmul(normal(1, (10, 72), bf)[:, 4:68], w, off), lambda: experts.grouped_matmul(x[:0], w, off, rows=rows),
        lambda: experts.grouped_matmul_dx(dy[:, :24], w, off), lambda: experts.grouped_matmul_dx(dy, w, off[1:]),
        lambda: experts.grouped_matmul_dw(dy, x[:9], off), lambda: experts.grouped_matmul_dw(dy, x, off, rows=rows[:9]),
        lambda: experts.grouped_matmul_dw(dy, x, off, dtype=torch.float16), lambda: experts.grouped_matmul_dw(dy, x.half(), off),
        lambda: experts.combine(z, slots.long()), lambda: experts.combine(z.float(), slots), lambda: experts.combine(z, slots, plan.weights[:, :1]),
        lambda: experts.combine(z.t(), slots), lambda: experts.combine_backward(dy, z, slots, None, off),
        lambda: experts.grad_norm([]), lambda: experts.grad_norm([z, z.cpu()]), lambda: experts.grad_norm([z.t()]), lambda: experts.grad_norm([slots]),
        lambda: experts.clip_grad_norm([z], -1.0), lambda: experts.clip_grad_norm([z], float("nan")), lambda: experts.clip_grad_norm([z], 1.0, out=[]),
        lambda: experts.clip_grad_norm([z], 1.0, out=[z[:3]]), lambda: experts.bind(len, z),
    ):
        with pytest.raises(FlexSpmvError):
            bad()
