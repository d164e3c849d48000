"""Vectors scale A x that leave float16's range, beside others that do not.

Bounds, whatever the scale: the vector is a sum of k products in 32 bits (k 2^-23 of their magnitudes), kept to 2^-22 of each value and 2^-17 of the largest of 32
neighbours; B's product adds (2 rank) 2^-23 of its magnitudes and 2 ^-23 of the whole, y's rounding half a step (2^-11, or half of the smallest step, 2^-25)."""
import numpy as np
import pytest
import torch

from flexspmv_b200 import adapters, experts

pytestmark = pytest.mark.gpu

FORMS = [(3, 128, 2048), (96, 264, 2048), (700, 264, 64), (1500, 1000, 264), (1700, 128, 72), (6000, 1000, 72), (1537, 128, 1472)]


def operands(tokens, n, k, rank, scales, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda shape: torch.randn(shape, generator=g, device="cuda")
    s = torch.tensor(scales, device="cuda")
    x, w, a = normal((tokens, k)).half(), (normal((n, k)) * k ** -0.5).half(), (normal((len(scales), rank, k)) * k ** -0.5).half()
    b = (normal((len(scales), n, rank)) * (0.3 / s[:, None, None])).clamp(-6e4, 6e4).half()
    return x, w, a, b, s


def check(y, x, w, a, b, scale, ids):
    x, w, ids = x.double(), w.double(), ids.long()
    k, rank = x.shape[1], a.shape[1]
    want, size = x @ w.t(), k * 2.0 ** -23 * (x.abs() @ w.abs().t())
    for i in range(a.shape[0]):
        t = torch.nonzero(ids == i).view(-1)
        s = float(scale[i].double())
        h, magnitudes = s * (x[t] @ a[i].double().t()), s * (x[t].abs() @ a[i].double().abs().t())
        largest = torch.nn.functional.pad(h.abs(), (0, -rank % 32)).view(t.numel(), (rank + 31) // 32, 32).amax(2).repeat_interleave(32, 1)[:, :rank]
        eh = (k + 1) * 2.0 ** -23 * magnitudes + 2.0 ** -22 * 1.01 * h.abs() + 2.0 ** -17 * 1.01 * largest
        bi = b[i].double().t()
        want[t] += h @ bi
        size[t] += eh @ bi.abs() + (2 * rank + 2) * 2.0 ** -23 * ((h.abs() + eh) @ bi.abs())
    bound = size + (2.0 ** -23 + 2.0 ** -11 * 1.01) * want.abs() + 2.0 ** -25 * 1.01
    err = (y.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, the worst by {float((err / bound).max()):.3g} bounds"


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 72, 128, 512])
@pytest.mark.parametrize("tokens,n,k", FORMS)
def test_vectors_beyond_a_float16(tokens, n, k, rank):
    scales = [1e5, 1.0, 2e-5, 3e6, 0.004, 65504.0 / 4]
    x, w, a, b, scale = operands(tokens, n, k, rank, scales)
    x[::7] *= 2.0 ** -9                                                       # tokens whose vectors are smaller
    r = np.random.default_rng(rank)
    runs = np.repeat(np.arange(30) % 7 - 1, r.integers(tokens // 12 + 1, tokens // 5 + 2, 30))[:tokens]
    for values in (np.arange(tokens) % 7 - 1, runs, np.full(tokens, 3), np.full(tokens, 2), np.full(tokens, 1)):
        ids = torch.from_numpy(values.astype(np.int32)).cuda()
        plan = adapters.plan(ids, len(scales))
        y = adapters.project(x, w, a, b, plan, scale=scale)
        check(y, x, w, a, b, scale, ids)
        assert torch.equal(adapters.project(x, w, a, b, plan, scale=scale), y)
    experts.check()


@pytest.mark.parametrize("tokens,n,k", FORMS)
def test_what_is_not_finite_stays_with_its_token(tokens, n, k):
    x, w, a, b, scale = operands(tokens, n, k, 40, [1e5, 1.0, 2e-5], seed=5)
    ids = torch.from_numpy((np.arange(tokens) * 3 // max(tokens, 1)).astype(np.int32)).cuda()
    plan = adapters.plan(ids, 3)
    want = adapters.project(x, w, a, b, plan, scale=scale)
    bad = x.clone()
    bad[0, 3], bad[tokens // 2, 0], bad[tokens - 1, k - 1] = float("inf"), float("nan"), float("-inf")
    got = adapters.project(bad, w, a, b, plan, scale=scale)
    others = torch.ones(tokens, dtype=torch.bool, device="cuda")
    others[[0, tokens // 2, tokens - 1]] = False
    assert torch.equal(got[others], want[others]) and not got[~others].isfinite().any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rank", [8, 24, 40])
@pytest.mark.parametrize("tokens,n,k", FORMS)
def test_an_infinite_scale(tokens, n, k, rank, dtype):
    """All else is positive: infinity, and not what infinity times the zeros beyond the rank would be."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w, a, b = (torch.rand(s, generator=g, device="cuda").add_(0.1).to(dtype) for s in ((tokens, k), (n, k), (2, rank, k), (2, n, rank)))
    ids = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    ids[tokens // 2:] = 1
    y = adapters.project(x, w, a, b, adapters.plan(ids, 2), scale=torch.tensor([float("inf"), 1e-3], device="cuda"))
    assert (y[ids == 0] == float("inf")).all() and y[ids == 1].isfinite().all()
