"""What a stack's dropout goes by: its own offset, or a seed that the caller gives; a pass that is run again for its gradients."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from flexspmv_b200 import residual
from flexspmv_b200.binding import FlexSpmvError
from flexspmv_b200.expert_layer import RoutedStack, Stacked

pytestmark = pytest.mark.gpu


def made():
    g = torch.Generator(device="cuda").manual_seed(4)
    stack = RoutedStack(64, 128, 8, 2, 3, p=0.3, generator=g, seed=11)
    return stack, torch.randn((120, 64), generator=g, device="cuda").to(torch.bfloat16)


def gradients(stack, out):
    (out.y.float().square().mean() + 0.01 * out.loss).backward()
    grads = [p.grad.clone() for p in stack.parameters()]
    stack.zero_grad(set_to_none=True)
    return grads


def test_a_given_seed():
    stack, x = made()
    own = stack(x)
    want = gradients(stack, own)
    assert stack.seed.tolist() == [11, 3]
    given = stack(x, seed=torch.tensor([11, 0], device="cuda"))
    assert torch.equal(given.y, own.y) and stack.seed.tolist() == [11, 3]
    assert all(torch.equal(a, b) for a, b in zip(gradients(stack, given), want))
    assert not torch.equal(stack(x, seed=torch.tensor([11, 1], device="cuda")).y, own.y)
    assert not torch.equal(stack(x, seed=torch.tensor([12, 0], device="cuda")).y, own.y)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_pass_that_is_run_again(reentrant):
    stack, x = made()
    seed = torch.tensor([5, 1 << 33], device="cuda")
    x = x.requires_grad_()
    want = gradients(stack, stack(x, seed=seed))
    again = Stacked(*checkpoint(stack, x, None, seed, use_reentrant=reentrant))          # reentrant: a plain tuple
    assert all(torch.equal(a, b) for a, b in zip(gradients(stack, again), want))
    out = Stacked(*checkpoint(stack, x, use_reentrant=reentrant))
    assert stack.seed[1] == 3
    with pytest.raises(FlexSpmvError, match="give forward a seed"):
        out.y.float().sum().backward()
    stack.zero_grad(set_to_none=True)
    stack.eval()                                        # nothing is dropped: any pass may be run again
    with torch.no_grad():
        want = stack(x).y
    out = Stacked(*checkpoint(stack, x, use_reentrant=reentrant))
    assert torch.equal(out.y, want)
    out.y.float().sum().backward()
    assert stack.shared[0].grad.any()


def test_layers_of_a_given_seed():
    """Layer i drops what its offset plus i says."""
    stack, x = made()
    seed = torch.tensor([7, 40], device="cuda")
    used = []
    plain = residual.layer_norm

    def watched(*args, **kwargs):
        if kwargs.get("seed") is not None:
            used.append(kwargs["seed"].tolist())
        return plain(*args, **kwargs)
    residual.layer_norm = watched
    try:
        stack(x, seed=seed)
    finally:
        residual.layer_norm = plain
    assert used == [[7, 40], [7, 41], [7, 42]]


def test_what_is_no_seed():
    stack, x = made()
    for bad in (torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int64), 5):
        with pytest.raises(FlexSpmvError, match="seed"):
            stack(x, seed=bad)
    stack.eval()
    with pytest.raises(FlexSpmvError, match="seed"):
        stack(x, seed=torch.zeros(1, dtype=torch.int64, device="cuda"))
