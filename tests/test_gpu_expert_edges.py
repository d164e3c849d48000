"""Where the expert operators' arguments leave the usual: rows of NaN, ids, ranges and sums at their ends.

Bounds as in ``test_gpu_experts``: n additions in 32 bits err by at most n * 2^-23 of the sum of magnitudes, one rounding to 16 bits by half a
unit (2^-8 of a bfloat16, 2^-11 of a float16); what is in whole numbers is equal."""
import gc
import shutil

import numpy as np
import pytest
import torch

from flexspmv_b200 import binding, experts
from flexspmv_b200.binding import FlexSpmvError
from flexspmv_b200.expert_layer import RoutedExperts

from test_gpu_experts import HALF, normal, offsets_of

pytestmark = pytest.mark.gpu

NEGATIVE_NAN = {torch.float32: (torch.int32, -0x400000), torch.bfloat16: (torch.int16, -0x40), torch.float16: (torch.int16, -0x200)}


# ---- router ------------------------------------------------------------------------------------------------------

def plain_route(logits, k):
    """The choice and the plan where NaN is never chosen: experts, offsets, rows, slots."""
    l = logits.double().cpu().numpy()
    l = np.where(np.isnan(l), -np.inf, l)
    tokens, n = l.shape
    ids = np.argsort(-l, axis=1, kind="stable")[:, :k]
    ids = np.where(np.isneginf(np.take_along_axis(l, ids, axis=1)), -1, ids)
    flat = ids.reshape(-1)
    pair = np.flatnonzero(flat >= 0)
    pair = pair[np.argsort(flat[pair], kind="stable")]
    rows, slots = np.full(flat.size, -1), np.full(flat.size, -1)
    rows[:pair.size] = pair // k
    slots[pair] = np.arange(pair.size)
    return ids, np.concatenate([[0], np.cumsum(np.bincount(flat[pair], minlength=n))]), rows, slots.reshape(tokens, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [8, 32, 60, 64, 128, 256, 384, 512, 1000, 1024])
def test_route_of_rows_of_nan(n, dtype):
    """Rows of NaN alone, of either sign, and rows with fewer than k other logits, among ordinary ones."""
    for tokens in (7, 41, 300):
        for k in (1, 8, min(n, 32)):
            clean = normal(n + tokens, (tokens, n), dtype)
            bad = torch.zeros((tokens, n), dtype=torch.bool, device="cuda")
            others = torch.rand((tokens, n), generator=torch.Generator(device="cuda").manual_seed(k), device="cuda").argsort(dim=1)
            for first, kept in ((1, 0), (2, 0), (3, k // 2), (4, k - 1), (5, k + 1)):          # of every six tokens the first is ordinary
                bad[first::6] = others[first::6] >= kept
            logits = clean.masked_fill(bad, float("nan"))
            as_int, pattern = NEGATIVE_NAN[dtype]
            logits[2::6] = torch.where(bad[2::6], torch.full_like(clean[2::6].view(as_int), pattern), clean[2::6].view(as_int)).view(dtype)
            logits[4::12, 0] = float("-inf")
            ids, offsets, rows, slots = plain_route(logits, k)
            spoiled = torch.isnan(logits).any(1).cpu().numpy()
            for renormalize in (False, True):
                plan = experts.route(logits, k, renormalize=renormalize)
                assert np.array_equal(plan.experts.cpu().numpy(), ids) and np.array_equal(plan.offsets.cpu().numpy(), offsets)
                assert np.array_equal(plan.rows.cpu().numpy(), rows) and np.array_equal(plan.slots.cpu().numpy(), slots)
                got = plan.weights.double().cpu().numpy()
                l = np.where(np.isnan(x := logits.double().cpu().numpy()), -np.inf, x)
                top = np.where(ids >= 0, np.take_along_axis(l, np.maximum(ids, 0), axis=1), -np.inf)
                base = np.where(np.isneginf(top[:, :1]), 0.0, top[:, :1])
                chosen, whole = np.exp(top - base), np.exp(l - base).sum(1, keepdims=True)
                total = chosen.sum(1, keepdims=True) if renormalize else whole
                want = chosen / np.where(total == 0, 1, total)
                if not renormalize:
                    want[spoiled] = np.where(ids[spoiled] >= 0, np.nan, 0.0)
                assert np.array_equal(np.isnan(got), np.isnan(want))
                assert np.all((np.abs(got - want) <= (n + 8) * 2.0 ** -23 * want + 1e-37) | np.isnan(want))
                # the gradient: rows without a choice are zeros, the other rows with NaN are NaN unless renormalized, and no row reaches another
                grad = experts.route_backward(torch.ones_like(plan.weights), logits, plan)
                none = torch.from_numpy(ids[:, 0] < 0)
                assert not grad[none.cuda()].any()
                lost = torch.from_numpy(spoiled) & ~none if not renormalize else torch.zeros_like(none)
                assert torch.equal(torch.isnan(grad).all(1).cpu(), lost) and torch.equal(torch.isnan(grad).any(1).cpu(), lost)
                ordinary = torch.arange(0, tokens, 6, device="cuda")
                alone = experts.route(clean[ordinary].contiguous(), k, renormalize=renormalize)
                assert torch.equal(plan.weights[ordinary], alone.weights)
                assert torch.equal(grad[ordinary], experts.route_backward(torch.ones_like(alone.weights), clean[ordinary].contiguous(), alone))


def test_route_backward_of_a_plan_of_other_logits():
    """Refused where the plan shows it; experts that the logits do not have are no choice, and nothing is written for them."""
    logits = normal(1, (50, 64), torch.float32)
    plan = experts.route(logits, 4)
    g = normal(2, (50, 4), torch.float32)
    with pytest.raises(FlexSpmvError, match="experts"):
        experts.route_backward(g, logits[:, :16].contiguous(), plan)
    for dtype, n in ((torch.float32, 64), (torch.bfloat16, 64), (torch.float16, 33)):
        logits = normal(3, (50, n), dtype)
        for renormalize in (False, True):
            plan = experts.route(logits, 4, renormalize=renormalize)
            want = experts.route_backward(torch.where(torch.arange(4, device="cuda") == 2, 0.0, g), logits,
                                          plan._replace(weights=plan.weights.clone(), experts=torch.where(torch.arange(4, device="cuda") == 2, -1, plan.experts)))
            for beyond in (n, n + 1, 2 ** 31 - 1, -2 ** 31):
                ids = torch.where(torch.arange(4, device="cuda") == 2, torch.full_like(plan.experts, beyond), plan.experts)
                around = torch.full((52, n), 7.0, dtype=dtype, device="cuda")
                got = experts.route_backward(g, logits, plan._replace(experts=ids), out=around[1:51])
                assert torch.equal(got, want) and bool((around[0] == 7.0).all()) and bool((around[51] == 7.0).all())
            all_beyond = plan._replace(experts=plan.experts + n)
            assert not experts.route_backward(g, logits, all_beyond).any()


# ---- the layer ---------------------------------------------------------------------------------------------------

def test_layer_frees_its_plans():
    """Steps of a training loop leave nothing behind, with Python's cyclic collector off."""
    layer = RoutedExperts(64, 128, 8, 2, generator=torch.Generator(device="cuda").manual_seed(1))
    x = normal(2, (3000, 64), torch.bfloat16)
    gc.collect()
    gc.disable()
    try:
        used = []
        for _ in range(6):
            layer(x).float().sum().backward()
            torch.cuda.synchronize()
            used.append(torch.cuda.memory_allocated())
        assert used[-1] == used[1]
    finally:
        gc.enable()


def test_tensors_that_require_a_gradient_are_refused():
    """Results of the operators carry none, so that one would be lost without a word; without recording they are taken."""
    bf = torch.bfloat16
    x, w, logits = normal(1, (10, 64), bf), normal(2, (3, 32, 64), bf), normal(3, (10, 3), torch.float32)
    plan = experts.route(logits, 2)
    y = experts.grouped_matmul(x, w, plan.offsets, rows=plan.rows)
    dy, dout, g = normal(4, (20, 32), bf), normal(5, (10, 32), bf), normal(6, (10, 2), torch.float32)
    r = lambda t: t.detach().requires_grad_()
    calls = [
        lambda f: experts.route(f(logits), 2), lambda f: experts.route_backward(f(g), logits, plan), lambda f: experts.route_backward(g, f(logits), plan),
        lambda f: experts.grouped_matmul(f(x), w, plan.offsets, rows=plan.rows), lambda f: experts.grouped_matmul(x, f(w), plan.offsets, rows=plan.rows),
        lambda f: experts.grouped_matmul_dx(f(dy), w, plan.offsets), lambda f: experts.grouped_matmul_dx(dy, f(w), plan.offsets),
        lambda f: experts.grouped_matmul_dw(f(dy), x, plan.offsets, rows=plan.rows), lambda f: experts.grouped_matmul_dw(dy, f(x), plan.offsets, rows=plan.rows),
        lambda f: experts.combine(f(y), plan.slots, plan.weights), lambda f: experts.combine(y, plan.slots, f(plan.weights)),
        lambda f: experts.combine_backward(f(dout), y, plan.slots, plan.weights, plan.offsets),
        lambda f: experts.combine_backward(dout, f(y), plan.slots, plan.weights, plan.offsets),
        lambda f: experts.bind(experts.combine, f(y), plan.slots),
    ]
    for call in calls:
        with pytest.raises(FlexSpmvError, match="gradient"):
            call(r)
        with torch.no_grad():
            call(r)
        call(lambda t: t)
    experts.check()


# ---- results in given memory -------------------------------------------------------------------------------------

def test_outputs_that_share_memory_with_inputs_are_refused():
    bf = torch.bfloat16
    x, w, logits = normal(1, (40, 64), bf), normal(2, (4, 64, 64), bf), normal(3, (40, 4), torch.float32)
    plan = experts.route(logits, 2)
    g = normal(4, (40, 2), torch.float32)
    rows, off = plan.rows[:40], offsets_of([7, 0, 20, 13])
    ones = torch.zeros((40, 1), dtype=torch.int32, device="cuda")
    wide = normal(5, (41, 128), bf)
    for bad in (
        lambda: experts.route_backward(g, logits, plan, out=logits), lambda: experts.grouped_matmul(x, w, off, out=x),
        lambda: experts.grouped_matmul(x[:39], w, off, out=x[1:]), lambda: experts.grouped_matmul(x, w, off, rows=rows, out=x),
        lambda: experts.grouped_matmul(x, w, off, out=w.view(-1, 64)[216:]), lambda: experts.grouped_matmul_dx(x, w, off, out=x),
        lambda: experts.grouped_matmul_dw(x, wide[:40, :64], off, out=wide.view(-1)[:4 * 64 * 64 // 4].view(1, 64, 64).expand(4, 64, 64)),
        lambda: experts.combine(x, ones, out=x), lambda: experts.bind(experts.grouped_matmul, x, w, off, out=x),
        lambda: experts.grouped_matmul(wide[:40, :64], w, off, out=wide.view(-1)[64:64 + 40 * 64].view(40, 64)),
    ):
        with pytest.raises(FlexSpmvError):
            bad()
    # beside the input, and between its rows, it may lie
    both = torch.cat([x, x])
    want = experts.grouped_matmul(x, w, off)
    assert torch.equal(experts.grouped_matmul(both[:40], w, off, out=both[40:]), want)
    assert torch.equal(experts.grouped_matmul(both[:40], w, off, out=both[40:]), want)
    one = torch.tensor([0, 1, 1, 1, 1], dtype=torch.int32, device="cuda")
    first = wide[:40, :64].clone()
    rows = torch.tensor([3], dtype=torch.int32, device="cuda")
    got = experts.grouped_matmul(wide[:40, :64], w, one, rows=rows, out=wide[7:8, 64:])
    assert torch.equal(got, experts.grouped_matmul(first, w, one, rows=rows)) and torch.equal(wide[:40, :64], first)
    experts.check()


def test_clip_of_tensors_that_share_memory():
    """A tensor given twice would be scaled once or twice, as its pieces come: refused.  Neighbours in one buffer are scaled each once."""
    flat = normal(1, (100_000,), torch.float32)
    a, b = flat[:40_000], flat[40_000:]
    for bad in (lambda: experts.clip_grad_norm([flat, flat], 1.0), lambda: experts.clip_grad_norm([flat, b], 1.0),
                lambda: experts.clip_grad_norm([a, b], 1.0, out=[b[:40_000], flat[:60_000].clone()]),
                lambda: experts.clip_grad_norm([flat[:50_000]], 1.0, out=[flat[4:50_004]]), lambda: experts.bind(experts.clip_grad_norm, [a, a], 1.0)):
        before = flat.clone()
        with pytest.raises(FlexSpmvError, match="share"):
            bad()
        assert torch.equal(flat, before)
    twice = float(experts.grad_norm([flat, flat]))                       # nothing is written: both count
    once = float(flat.double().norm())
    assert abs(twice - 2 ** 0.5 * once) <= 1e-5 * once
    before = flat.clone()
    norm = experts.clip_grad_norm([b, a], 1.0)
    assert abs(float(norm) - once) <= 1e-5 * once and torch.allclose(flat, before / (once + 1e-6), rtol=1e-5, atol=0)


def test_clip_is_not_bound_inside_a_capture():
    """Its plan would only be recorded.  The plain call in a capture is, plan and all, and follows the tensors."""
    ts = [normal(1, (5000,), torch.bfloat16), normal(2, (77,), torch.float32)]
    outs = [torch.zeros(t.shape, device="cuda") for t in ts]
    experts.clip_grad_norm(ts, 1.0, out=outs)
    torch.cuda.synchronize()
    for bind in (lambda: experts.bind(experts.clip_grad_norm, ts, 1.0, out=outs), lambda: experts.bind(experts.grad_norm, ts)):
        refused = []
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            try:
                bind()
            except FlexSpmvError as e:
                refused.append(str(e))
            norm = experts.clip_grad_norm(ts, 1.0, out=outs)
        assert len(refused) == 1 and "captured" in refused[0]
        for _ in range(2):
            for t in ts:
                t.mul_(2)
            graph.replay()
            exact = sum(float((t.double() ** 2).sum()) for t in ts) ** 0.5
            assert abs(float(norm) - exact) <= 1e-5 * exact
            assert all(torch.allclose(o, t.float() / (exact + 1e-6), rtol=1e-5) for o, t in zip(outs, ts))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_of_values_whose_squares_leave_32_bits(dtype):
    """Finite gradients have a finite norm as far as 32 bits hold it.  A thread adds at most 256 squares, in 32 bits or in 64, and the rest in 64:
    256 * 2^-24 and a square root's rounding."""
    tol = 300 * 2.0 ** -24
    for scales in ([1e20], [1e-25], [3e37, 1.0], [1e-30, 1e-38], [2e18, 1e18], [1e-22, 0.0], [1e-19, 1e-19], [1e20, 1e-25, 1.0, 0.0], [0.0]):
        for length in (1, 4099, 300_001):
            ts = [normal(i, (length + i,), torch.float32).mul_(s * (0.1 if s > 1e30 else 1.0)).to(dtype)[i % 2:] for i, s in enumerate(scales)]
            exact = sum(float((t.double() ** 2).sum()) for t in ts) ** 0.5
            if exact > 3e38:
                continue
            norm = experts.grad_norm(ts)
            assert abs(float(norm) - exact) <= tol * exact, (scales, length)
            for max_norm in (1.0, exact / 3):
                if max_norm == 0.0:
                    continue
                mine = [t.clone() for t in ts]
                assert torch.equal(experts.clip_grad_norm(mine, max_norm), norm)
                scale = min(1.0, max_norm / (exact + 1e-6))
                half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
                # below the types' normal range a rounding is up to half of their smallest value, 2^-149 or 2^-133; the scale, too, is held in 32 bits
                low = 2.0 ** -149 if dtype == torch.float32 else 2.0 ** -133
                for t, m in zip(ts, mine):
                    want = t.double() * scale
                    bound = (1.01 * half + tol + 2.0 ** -22 + 2.0 ** -149 / scale) * want.abs() + low
                    assert bool(((m.double() - want).abs() <= bound).all()), (scales, length, max_norm)
    beyond = [torch.full((300_000,), 3e38, device="cuda").to(dtype)]
    assert float(experts.grad_norm(beyond)) == float("inf")


# ---- logits far apart --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k", [(2, 2), (8, 8), (16, 4), (64, 32), (300, 32)])
def test_route_of_logits_far_apart(n, k, dtype):
    """Weights to the bound that near logits have, (n + 8) * 2^-23 of each, however small: a power of a difference as rounded would be off by as many
    units as the difference has.  The sum's terms count by what they are, so that their powers' d * 2^-23 stays below one of its n units."""
    for tokens in (5, 700):
        logits = (torch.rand((tokens, n), generator=torch.Generator(device="cuda").manual_seed(n), device="cuda") * 80 - 40).to(dtype)
        logits[0] = torch.linspace(-40.1, 39.7, n, device="cuda").to(dtype)
        logits[1] = torch.linspace(0.3, -79.9, n, device="cuda").to(dtype)
        l = logits.double().cpu().numpy()
        ids = np.argsort(-l, axis=1, kind="stable")[:, :k]
        for renormalize in (False, True):
            plan = experts.route(logits, k, renormalize=renormalize)
            assert np.array_equal(plan.experts.cpu().numpy(), ids)
            e = np.exp(l - l.max(1, keepdims=True))
            top = np.take_along_axis(e, ids, axis=1)
            want = top / (top if renormalize else e).sum(1, keepdims=True)
            assert np.all(np.abs(plan.weights.double().cpu().numpy() - want) <= (n + 8) * 2.0 ** -23 * want + 1e-37)
            g = normal(7, (tokens, k), torch.float32)
            got = experts.route_backward(g, logits, plan).double().cpu().numpy()
            p, gd = e / e.sum(1, keepdims=True), np.zeros_like(l)
            np.put_along_axis(gd, ids, g.double().cpu().numpy(), axis=1)
            gw = np.take_along_axis(gd, ids, axis=1) * want
            mean, size = gw.sum(1, keepdims=True), np.abs(gw).sum(1, keepdims=True)
            if renormalize:
                p = np.zeros_like(l)
                np.put_along_axis(p, ids, want, axis=1)
            bound = (n + k + 24) * 2.0 ** -23 * p * (np.abs(gd) + size) + 1e-37
            if dtype != torch.float32:                 # one rounding, and float16's smallest values
                bound += HALF[dtype] * 1.01 * np.abs(p * (gd - mean)) + (2.0 ** -25 if dtype == torch.float16 else 0)
            assert np.all(np.abs(got - p * (gd - mean)) <= bound)


# ---- long sums ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,counts,n,k", [
    (torch.float16, [600_000], 72, 64),                        # a cluster divides the sum
    (torch.float16, [3, 70_000, 0, 600_000, 65_536, 65_600, 1], 136, 264),
    (torch.float16, [200_000, 17], 2048, 1024),                # tiles that go round the pairs
    (torch.bfloat16, [4_000_000], 72, 64),
    (torch.bfloat16, [100, 3_000_000], 520, 8),
    (torch.float16, [16_384, 16_448, 40, 8000], 264, 136),
])
def test_dw_in_16_bits_over_many_rows(dtype, counts, n, k):
    """Rows of one sign, of which the matrix instructions' cut sums fall short the more the longer they are.  With more than 16 384 (131 072) rows all
    sums are in parts of 4096: 256 instructions that cut two units at most, then the parts' correctly rounded additions."""
    slots = sum(counts)
    g = torch.Generator(device="cuda").manual_seed(slots)
    x, dy = torch.empty((slots, k), dtype=dtype, device="cuda"), torch.empty((slots, n), dtype=dtype, device="cuda")
    for at in range(0, slots, 100_000):
        x[at:at + 100_000] = torch.rand(x[at:at + 100_000].shape, generator=g, device="cuda") + 0.5
        dy[at:at + 100_000] = (torch.rand(dy[at:at + 100_000].shape, generator=g, device="cuda") + 0.5) * 2.0 ** -8
    dw = experts.grouped_matmul_dw(dy, x, offsets_of(counts))
    experts.check()
    long = 16_384 if dtype == torch.float16 else 131_072
    at, columns = 0, slice(0, 64)
    for e, c in enumerate(counts):
        want = torch.zeros((n, min(k, 64)), dtype=torch.float64, device="cuda")
        for b in range(at, at + c, 100_000):
            rows = slice(b, min(b + 100_000, at + c))
            want += dy[rows].double().t() @ x[rows, columns].double()
        at += c
        got = dw[e, :, columns].double()
        cut = (512 + c / 8192 if c > long else c) * 2.0 ** -23
        low = 2.0 ** -25 if dtype == torch.float16 else 0.0
        assert bool(((got - want).abs() <= (cut + 1.01 * HALF[dtype]) * want + low).all()), (e, c)


def test_layer_where_masked_tokens_hold_anything():
    """NaN and infinity in tokens that the mask leaves out reach neither the result nor a gradient."""
    layer = RoutedExperts(64, 128, 8, 2, generator=torch.Generator(device="cuda").manual_seed(1))
    clean = normal(2, (300, 64), torch.bfloat16)
    mask = torch.rand(300, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") < 0.7
    dirty = clean.clone()
    dirty[~mask] = float("nan")
    dirty[torch.nonzero(~mask)[0]] = float("inf")
    dy = normal(4, (300, 64), torch.bfloat16)
    results = []
    for x in (clean, dirty):
        x = x.clone().requires_grad_()
        layer.zero_grad()
        y = layer(x, mask)
        y.backward(dy)
        results.append([y.detach(), x.grad] + [p.grad.clone() for p in layer.parameters()])
    experts.check()
    assert not results[1][0][~mask].any() and not results[1][1][~mask].any()
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_two_copies_of_the_library(tmp_path, monkeypatch):
    """load_library takes a path: each copy in a process asks for its own kernels' shared memory."""
    x, w, off = normal(1, (300, 256), torch.bfloat16), normal(2, (3, 128, 256), torch.bfloat16), offsets_of([100, 0, 200])
    logits = normal(3, (5000, 256), torch.float32)
    want = experts.grouped_matmul(x, w, off), experts.route(logits, 8).slots
    path = str(shutil.copy(binding.DEFAULT_LIB, tmp_path / "copy.so"))
    lib = binding.load_library(path)
    monkeypatch.setattr(experts, "load_library", lambda: lib)
    monkeypatch.setattr(experts, "_functions", {})
    assert torch.equal(experts.grouped_matmul(x, w, off), want[0]) and torch.equal(experts.route(logits, 8).slots, want[1])
    experts.check()


def test_clip_asked_to_write_by_a_plan_for_the_norm_alone():
    t = normal(1, (100_000,), torch.float32)
    before = t.clone()
    call = experts.bind(experts.grad_norm, [t])
    want = float(call.launch())
    pieces, _, _, *rest = call._args                      # C arguments: pieces, write, max_norm, norm, workspace, its bytes
    call._args = (pieces, 1, 0.5, *rest)
    assert float(call.launch()) == want and torch.equal(t, before)
