"""Plans that do not fit the call: nothing is read or written out of range, and the call is an error.

Each plan here has numbers that the kernels' own checks reject: other tokens or adapters, tiles and rows out of range."""
import numpy as np
import pytest
import torch

from flexspmv_b200 import adapters, experts
from flexspmv_b200.binding import FlexSpmvError

pytestmark = pytest.mark.gpu


def operands(tokens, n=264, k=136, count=5, rank=16, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x, w, a, b = (torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((tokens, k), (n, k), (count, rank, k), (count, n, rank)))
    return x, w, a, b, torch.from_numpy((np.arange(tokens) % (count + 1) - 1).astype(np.int32)).cuda()


def refused(x, w, a, b, plan, good):
    """The call leaves an error, the next one with a plan that fits is as it was."""
    want = adapters.project(x, w, a, b, good)
    experts.check()
    room = torch.full((x.shape[0] + 2, w.shape[0]), 7.0, dtype=x.dtype, device="cuda")
    adapters.project(x, w, a, b, plan, out=room[1:-1])
    with pytest.raises(FlexSpmvError, match="rows or ids"):
        experts.check()
    assert (room[0] == 7).all() and (room[-1] == 7).all()
    assert torch.equal(adapters.project(x, w, a, b, good), want)
    experts.check()


@pytest.mark.parametrize("rank", [16, 128])
@pytest.mark.parametrize("tokens", [1, 40, 700, 2000, 5000])
def test_plans_that_are_not_there_yet(tokens, rank):
    x, w, a, b, ids = operands(tokens, rank=rank)
    good = adapters.plan(ids, 5)
    plan = experts.bind(adapters.plan, ids, 5).outputs
    for fill in (0, -1, 0x3fffffff, -0x40000000):
        plan.data.fill_(fill)
        refused(x, w, a, b, plan, good)


@pytest.mark.parametrize("tokens", [1, 40, 700, 2000])
def test_numbers_out_of_range(tokens):
    """A plan of these tokens and adapters, of which tiles or rows leave their arrays."""
    x, w, a, b, ids = operands(tokens)
    good = adapters.plan(ids, 5)
    count = int(good.data[0])
    if tokens == 1:                                     # its only token has no adapter
        good = adapters.plan(ids + 1, 5)
        count = 1
    assert count >= 1 and good.data[1:3].tolist() == [tokens, 5]
    last = 8 + 4 * (count - 1)                          # the last tile: adapter, first place, places
    for at, value in ((last, 5), (last, -1), (last, 1 << 30), (last + 1, tokens), (last + 1, -1), (last + 1, -(1 << 31)), (last + 1, (1 << 31) - 1),
                      (last + 2, 17), (last + 2, 0), (last + 2, -5), (last + 2, 1 << 30)):
        data = good.data.clone()
        data[at] = value
        refused(x, w, a, b, good._replace(data=data), good)
    # rows: the places are those of the tiles, `rows` lies behind the ids
    tiles = tokens // 16 + min(tokens, 5)
    rows = 8 + 4 * tiles + 6 + tokens
    for value in (tokens, -1, 1 << 30, -(1 << 31)):
        data = good.data.clone()
        data[rows] = value
        refused(x, w, a, b, good._replace(data=data), good)


def test_plans_of_other_batches():
    """As a caller of the C interface may give them: of other tokens, of other adapters, in room for either."""
    x, w, a, b, ids = operands(300)
    good = adapters.plan(ids, 5)
    few = ids.clamp(max=3)
    for other in (adapters.plan(ids[:200], 5), adapters.plan(few, 4), adapters.plan(few[:299], 4)):
        data = torch.zeros_like(good.data)
        n = min(data.numel(), other.data.numel())
        data[:n] = other.data[:n]
        refused(x, w, a, b, adapters.Plan(data, 300, 5), good)
