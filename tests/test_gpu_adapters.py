"""Low-rank adapters beside a shared projection (``flexspmv_b200.adapters``) against the formula in 64 bits.

Bounds.  A sum of n products in 32 bits is off by at most n * 2^-23 of the products' magnitudes (a matrix instruction cuts what an addition rounds).  scale A x is
kept to 2^-17 (bfloat16) or 2^-22 and half of float16's smallest step (2^-25), and enters y through B.  One rounding to 16 bits is added."""
import numpy as np
import pytest
import torch

from flexspmv_b200 import adapters, experts
from flexspmv_b200.binding import FlexSpmvError

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
KEPT = {torch.bfloat16: (2.0 ** -17, 0.0), torch.float16: (2.0 ** -22, 2.0 ** -25)}


def normal(seed, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale).to(dtype)


def operands(tokens, n, k, count, rank, dtype, seed=0):
    return (normal(seed, (tokens, k), dtype), normal(seed + 1, (n, k), dtype, k ** -0.5), normal(seed + 2, (count, rank, k), dtype, k ** -0.5),
            normal(seed + 3, (count, n, rank), dtype, 0.3), torch.rand(count, generator=torch.Generator(device="cuda").manual_seed(seed + 4), device="cuda") + 0.5)


def ids_of(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def check(y, x, w, a, b, ids, scale):
    x, w, ids = x.double(), w.double(), ids.long()
    k, rank = x.shape[1], a.shape[1]
    want, size = x @ w.t(), k * 2.0 ** -23 * (x.abs() @ w.abs().t())
    rel, low = KEPT[y.dtype]
    for i in torch.unique(ids).tolist():
        if i < 0:
            continue
        t = torch.nonzero(ids == i).view(-1)
        s = float(scale[i].double()) if scale is not None else 1.0
        h, ah = s * (x[t] @ a[i].double().t()), s * (x[t].abs() @ a[i].double().abs().t())
        eh = (k + 1) * 2.0 ** -23 * ah + rel * h.abs() * 1.01 + low
        bi = b[i].double().t()
        want[t] += h @ bi
        size[t] += eh @ bi.abs() + (2 * rank + 2) * 2.0 ** -23 * ((h.abs() + eh) @ bi.abs())
    # the two parts' sum, and the only rounding
    bound = size + 2.0 ** -23 * want.abs() + HALF[y.dtype] * want.abs() * 1.01 + (2.0 ** -24 if y.dtype == torch.float16 else 0.0) + 1e-30
    err = (y.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, the worst by {float((err / bound).max()):.3g} bounds"


def patterns(tokens, count, seed=0):
    r = np.random.default_rng([tokens, count, seed])
    yield np.full(tokens, -1)
    yield np.full(tokens, count - 1)
    yield np.arange(tokens) % count
    yield r.integers(-1, count, tokens)
    runs = np.repeat(r.integers(-1, count, tokens), r.integers(1, 40, tokens))[:tokens]
    yield runs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,n,k,count,rank", [
    (1, 8, 8, 1, 8), (1, 4096, 2048, 3, 16), (2, 136, 72, 4, 16), (7, 1000, 1416, 5, 24), (16, 64, 64, 2, 8), (17, 128, 4096, 40, 32), (48, 4096, 4096, 64, 16),
    (48, 520, 264, 64, 40), (64, 256, 512, 9, 64), (65, 1032, 200, 70, 72), (200, 384, 1000, 200, 128), (513, 4096, 256, 30, 8), (1024, 512, 512, 3, 48),
    (1025, 520, 520, 1024, 16), (1031, 1000, 1416, 96, 8), (2500, 2048, 1024, 20, 64), (5000, 264, 136, 7, 256), (300, 136, 264, 3, 512), (300, 4096, 4096, 20, 16), (130, 2048, 2048, 40, 32), (150, 1000, 6000, 64, 128), (3000, 512, 264, 5, 24), (2100, 520, 1000, 3, 40),
    (1500, 264, 264, 4, 72), (4097, 136, 72, 300, 16)])
def test_project(tokens, n, k, count, rank, dtype):
    x, w, a, b, scale = operands(tokens, n, k, count, rank, dtype)
    for i, values in enumerate(patterns(tokens, count)):
        ids = ids_of(values)
        plan = adapters.plan(ids, count)
        y = adapters.project(x, w, a, b, plan, scale=scale if i % 2 else None)
        check(y, x, w, a, b, ids, scale if i % 2 else None)
    experts.check()
    # the same bits again, with rows apart
    room = torch.full((tokens, k + 8), float("nan"), dtype=dtype, device="cuda")
    room[:, :k] = x
    assert torch.equal(adapters.project(room[:, :k], w, a, b, plan), y if i % 2 == 0 else adapters.project(x, w, a, b, plan))


@pytest.mark.parametrize("tokens,n,k,count,rank", [(8192, 4096, 2048, 12, 64), (12000, 2048, 4096, 100, 16)])
def test_project_large(tokens, n, k, count, rank):
    x, w, a, b, scale = operands(tokens, n, k, count, rank, torch.bfloat16)
    for values in list(patterns(tokens, count))[2:]:
        ids = ids_of(values)
        check(adapters.project(x, w, a, b, adapters.plan(ids, count), scale=scale), x, w, a, b, ids, scale)


def test_so_many_tokens_that_groups_are_longer_runs():
    """More than 64 000 tokens: at most some 1000 groups, and runs around their limit."""
    tokens, n, k, count, rank = 150_000, 72, 64, 50, 16
    x, w, a, b, scale = operands(tokens, n, k, count, rank, torch.bfloat16)
    r = np.random.default_rng(3)
    for lengths in (r.integers(1, 700, 1000), np.full(600, 299), np.full(600, 300), r.integers(1, 3, 110_000)):
        ids = np.repeat(np.arange(lengths.size) * 7 % (count + 1) - 1, lengths)[:tokens]
        ids = ids_of(np.concatenate([ids, np.full(tokens - ids.size, 2)]))
        check(adapters.project(x, w, a, b, adapters.plan(ids, count), scale=scale), x, w, a, b, ids, scale)
    experts.check()


@pytest.mark.parametrize("tokens", [1100, 3000])
def test_runs_around_the_length_of_a_group(tokens):
    n, k, count, rank = 520, 136, 9, 40
    x, w, a, b, scale = operands(tokens, n, k, count, rank, torch.float16)
    for lengths in ([127, 128, 129, 1, 128, 64, 64, 200, 1, 1], [1] * 10 + [128] * 3 + [5] + [300], [tokens], [tokens - 1, 1], [1, tokens - 1]):
        values = np.resize(np.repeat(np.arange(len(lengths)) % (count + 1) - 1, lengths), tokens)
        ids = ids_of(values)
        check(adapters.project(x, w, a, b, adapters.plan(ids, count), scale=scale), x, w, a, b, ids, scale)


@pytest.mark.parametrize("tokens,n,k,rank", [(5, 136, 264, 16), (48, 512, 512, 32), (300, 512, 264, 16), (3000, 1024, 512, 64), (300, 4096, 512, 128)])
def test_an_adapter_reaches_its_own_tokens_only(tokens, n, k, rank):
    """NaN and infinity in one adapter, in one token and in adapters that nobody has: every other token as without."""
    count = 6
    x, w, a, b, scale = operands(tokens, n, k, count, rank, torch.bfloat16)
    ids = ids_of(np.random.default_rng(1).integers(-1, 4, tokens))
    ids[0], ids[1], ids[2] = 2, 0, -1
    want = adapters.project(x, w, a, b, adapters.plan(ids, count), scale=scale)
    a2, b2, s2, x2 = a.clone(), b.clone(), scale.clone(), x.clone()
    a2[4:], b2[4:], s2[4:] = float("nan"), float("inf"), float("nan")
    b2[2] = float("inf")
    b2[2, ::2] = float("nan")
    a2[3, 0, 0] = float("inf")
    x2[1] = float("nan")
    got = adapters.project(x2, w, a2, b2, adapters.plan(ids, count), scale=s2)
    good = (ids != 2) & (ids != 3)
    good[1] = False
    assert torch.equal(got[good], want[good])
    assert not got[ids == 2].isfinite().any() and got[1].isnan().all()


def test_a_long_run_keeps_to_itself():
    """Groups of one adapter each, one of them infinite and one not a number, between others and tokens without any."""
    tokens, n, k, count, rank = 2000, 520, 264, 6, 24
    x, w, a, b, scale = operands(tokens, n, k, count, rank, torch.bfloat16)
    ids = ids_of(np.repeat([0, 2, 1, -1, 3, 0, 2, 1], [300, 250, 150, 333, 267, 40, 260, 400]))
    want = adapters.project(x, w, a, b, adapters.plan(ids, count), scale=scale)
    a2, b2, s2 = a.clone(), b.clone(), scale.clone()
    b2[2], a2[3] = float("inf"), float("nan")
    s2[3:] = float("nan")
    got = adapters.project(x, w, a2, b2, adapters.plan(ids, count), scale=s2)
    bad = (ids == 2) | (ids == 3)
    assert torch.equal(got[~bad], want[~bad]) and not got[bad].isfinite().any()


def test_more_precise_than_a_16_bit_vector():
    """W x and B A x cancel: what is left shows scale A x to more than 16 bits."""
    for tokens in (3, 96, 700, 1500):                                        # the divided, the mixed and the grouped form
        n, k, rank = 256, 512, 16
        x, w, a, b, _ = operands(tokens, n, k, 2, rank, torch.bfloat16)
        w = (-(b[1].double() @ a[1].double())).bfloat16()
        ids = ids_of(np.full(tokens, 1))
        check(adapters.project(x, w, a, b, adapters.plan(ids, 2)), x, w, a, b, ids, None)


def test_a_bound_plan_follows_its_ids_in_a_graph():
    count, rank, n, k = 16, 16, 1024, 512
    for tokens in (12, 400, 3000):
        x, w, a, b, scale = operands(tokens, n, k, count, rank, torch.bfloat16)
        ids = ids_of(np.zeros(tokens))
        plan = experts.bind(adapters.plan, ids, count)
        one, two = (experts.bind(adapters.project, x, m, a, b, plan.outputs, scale=scale) for m in (w, w * 2))
        for c in (plan, one, two):
            c.launch()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.launch(), one.launch(), two.launch()
        for i, values in enumerate(patterns(tokens, count)):
            ids.copy_(ids_of(values))
            x.copy_(normal(50 + i, x.shape, x.dtype))
            graph.replay()
            check(one.outputs, x, w, a, b, ids, scale)
            check(two.outputs, x, w * 2, a, b, ids, scale)
    experts.check()


def test_back_to_back_launches_follow_their_inputs():
    """Each launch reads what the launch before it wrote: no load runs ahead of the kernel that fills x."""
    width, count = 512, 4
    x, w, a, b, scale = operands(40, width, width, count, 16, torch.bfloat16)
    plan = adapters.plan(ids_of(np.arange(40) % 5 - 1), count)
    first = adapters.project(x, w, a, b, plan, scale=scale)
    second = adapters.project(first, w, a, b, plan, scale=scale)
    third = adapters.project(second, w, a, b, plan, scale=scale)
    torch.cuda.synchronize()
    buf = [torch.empty_like(first) for _ in range(3)]
    for _ in range(20):
        y = x
        for t in buf:
            y = adapters.project(y, w, a, b, plan, scale=scale, out=t)
    assert all(torch.equal(p, q) for p, q in zip(buf, (first, second, third)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = adapters.project(first, w, a, b, plan, scale=scale)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, second)


def test_two_streams_at_once():
    """Calls of two batches on two streams, each two launches of which the second begins early."""
    sides = [torch.cuda.Stream() for _ in range(2)]
    calls, want = [], []
    for i, tokens in enumerate((48, 2000)):
        x, w, a, b, scale = operands(tokens, 1024, 1024, 8, 32, torch.bfloat16, seed=10 * i)
        ids = ids_of(np.sort(np.random.default_rng(i).integers(-1, 8, tokens)))
        plan = adapters.plan(ids, 8)
        want.append(adapters.project(x, w, a, b, plan, scale=scale))
        check(want[-1], x, w, a, b, ids, scale)
        calls.append(experts.bind(adapters.project, x, w, a, b, plan, scale=scale))
    torch.cuda.synchronize()
    for _ in range(30):
        for side, call in zip(sides, calls):
            with torch.cuda.stream(side):
                call.launch()
    torch.cuda.synchronize()
    for call, exact in zip(calls, want):
        assert torch.equal(call.outputs, exact)
    experts.check()


def test_ids_that_are_no_adapter_are_noticed():
    x, w, a, b, _ = operands(20, 64, 64, 3, 8, torch.bfloat16)
    values = np.arange(20) % 4 - 1
    want = adapters.project(x, w, a, b, adapters.plan(ids_of(values), 3))
    bad = values.copy()
    bad[values < 0] = 7
    bad[0] = -5
    plan = adapters.plan(ids_of(bad), 3)
    torch.cuda.synchronize()
    with pytest.raises(FlexSpmvError, match="ids"):
        adapters.project(x, w, a, b, plan)
    assert torch.equal(adapters.project(x, w, a, b, plan), want)          # they counted as none
    experts.check()


def test_refusals():
    x, w, a, b, scale = operands(20, 64, 72, 3, 8, torch.bfloat16)
    ids = ids_of(np.zeros(20))
    plan = adapters.plan(ids, 3)
    for call in (lambda: adapters.plan(ids.long(), 3), lambda: adapters.plan(ids, 0), lambda: adapters.plan(ids, 1025), lambda: adapters.plan(ids[::2], 3),
                 lambda: adapters.project(x, w, a, b, adapters.plan(ids[:5], 3)), lambda: adapters.project(x, w, a, b, adapters.plan(ids, 4)),
                 lambda: adapters.project(x.half(), w, a, b, plan), lambda: adapters.project(x, w[:, :64], a, b, plan),
                 lambda: adapters.project(x, w[:60], a, b[:, :60].contiguous(), plan), lambda: adapters.project(x, w, a[:, :4].contiguous(), b[..., :4].contiguous(), plan),
                 lambda: adapters.project(x, w, a, b[:2], plan), lambda: adapters.project(x, w, a, b.transpose(1, 2), plan),
                 lambda: adapters.project(x, w, a, b, plan, scale=scale[:2]), lambda: adapters.project(x, w, a, b, plan, scale=scale.half()),
                 lambda: adapters.project(x, w, a, b, plan, out=x), lambda: adapters.project(x, w, a, b, ids), lambda: adapters.project(x.t(), w, a, b, plan),
                 lambda: adapters.project(x, w.detach().requires_grad_(), a, b, plan), lambda: adapters.project(x[:, 1:65], w, a, b, plan)):
        with pytest.raises(FlexSpmvError):
            call()
    assert adapters.project(x[:0], w, a, b, adapters.plan(ids[:0], 3)).shape == (0, 64)
