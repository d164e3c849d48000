"""The vector scale A x of an adapter, between its two products, is the sum of 32 bits that it is.

Bounds.  Where y is a power of two that sums of 32 bits reach without an error it is that value."""
import numpy as np
import pytest
import torch

from flexspmv_b200 import adapters, experts

pytestmark = pytest.mark.gpu

# The forms of the second product: tiles that CTAs divide, and that they do not; of one adapter, whose part is steps of the same sum, narrow and wide, and divided.
FORMS = [(3, 128, 2048), (96, 128, 2048), (700, 264, 64), (1500, 1000, 264), (1700, 128, 72), (9000, 1000, 72), (1537, 128, 1472)]


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 128, 512])
@pytest.mark.parametrize("tokens,n,k", FORMS)
def test_bits_of_the_vector(tokens, n, k, rank):
    """The first value of the vector is 1 + 2^-9 + 2^-18 (for float16 2^-21), the next two -1 and -2^-9: only the last of its bits is left in y."""
    for dtype, last in ((torch.bfloat16, 2.0 ** -18), (torch.float16, 2.0 ** -21)):
        x = torch.zeros((tokens, k), dtype=dtype, device="cuda")
        x[:, 1], x[:, k - 8], x[:, k - 1] = 1.0, 2.0 ** -9, last
        a = torch.zeros((2, rank, k), dtype=dtype, device="cuda")
        first, second, third = 5, rank - 1, rank // 2
        a[1, first, 1] = a[1, first, k - 8] = a[1, first, k - 1] = 1.0
        a[1, second, 1], a[1, third, k - 8] = -1.0, -1.0
        b = torch.zeros((2, n, rank), dtype=dtype, device="cuda")
        b[1, :, first] = b[1, :, second] = b[1, :, third] = 1.0
        w = torch.zeros((n, k), dtype=dtype, device="cuda")
        ids = torch.from_numpy(np.full(tokens, 1, dtype=np.int32)).cuda()
        y = adapters.project(x, w, a, b, adapters.plan(ids, 2))
        assert torch.equal(y, torch.full_like(y, last))
    experts.check()


def test_divided_sums_that_begin_with_the_vector():
    """A long rank beside a short sum, in runs of one adapter: a CTA's share of the divided sum is the vector's steps alone.  The same bits twice, after
    another product has left its sums where they are made."""
    tokens, n, k, rank = 1537, 128, 1472, 512
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = (torch.randn(s, generator=g, device="cuda").to(torch.bfloat16) for s in ((tokens, k), (n, k)))
    a, b = (torch.randn(s, generator=g, device="cuda").mul_(k ** -0.5).to(torch.bfloat16) for s in ((3, rank, k), (3, n, rank)))
    ids = torch.from_numpy(np.repeat([0, 1, 2], [512, 512, 513]).astype(np.int32)).cuda()
    plan = adapters.plan(ids, 3)
    y = adapters.project(x, w, a, b, plan)
    experts.grouped_matmul(x.mul(100.0), w.mul(100.0)[None], torch.tensor([0, tokens], dtype=torch.int32, device="cuda"))
    assert torch.equal(adapters.project(x, w, a, b, plan), y)
    h = torch.einsum("tk,trk->tr", x.double(), a.double()[ids.long()])
    want = x.double() @ w.double().t() + torch.einsum("tr,tnr->tn", h, b.double()[ids.long()])
    size = x.double().abs() @ w.double().abs().t() + torch.einsum("tr,tnr->tn", h.abs(), b.double().abs()[ids.long()])
    # an error of n 2^-23 of the products' magnitudes in each sum of n, of the vector's through B, and y's rounding
    eh = torch.einsum("tk,trk->tr", x.double().abs(), a.double().abs()[ids.long()]) * k * 2.0 ** -23
    bound = (k + 3 * rank) * 2.0 ** -23 * size + torch.einsum("tr,tnr->tn", eh, b.double().abs()[ids.long()]) + 2.0 ** -8 * 1.01 * want.abs()
    assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,n,k,rank", [(48, 264, 200, 16), (48, 264, 200, 40), (40, 128, 2048, 16), (40, 128, 2048, 64), (700, 264, 64, 8), (700, 1000, 72, 72)])
def test_a_token_gets_the_same_bits_whoever_shares_its_adapter(tokens, n, k, rank, dtype):
    """One, two, some or all of the others, in a row or scattered, with the adapter's own weights under another number."""
    g = torch.Generator(device="cuda").manual_seed(6)
    x, w, a, b = (torch.randn(s, generator=g, device="cuda").mul_(0.3).to(dtype) for s in ((tokens, k), (n, k), (8, rank, k), (8, n, rank)))
    a[1:] = a[0]
    b[1:] = b[0]
    base = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    want = adapters.project(x, w, a, b, adapters.plan(base, 8))
    r = np.random.default_rng(1)
    for values in (np.arange(tokens) % 8, np.arange(tokens) // 2 % 8, np.arange(tokens) // 3 % 8, np.arange(tokens) // 5 % 8, r.integers(0, 8, tokens), r.integers(0, 8, tokens) // 6,
                   r.integers(0, 8, tokens) // 7):
        ids = torch.from_numpy(values.astype(np.int32)).cuda()
        assert torch.equal(adapters.project(x, w, a, b, adapters.plan(ids, 8)), want)
