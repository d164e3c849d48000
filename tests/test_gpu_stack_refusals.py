"""What the decoding classes of ``expert_layer`` refuse."""
import pytest
import torch

from flexspmv_b200.binding import FlexSpmvError
from flexspmv_b200.expert_layer import Adapter, DecodingStack, DecodingStep, RoutedExperts, RoutedStack

pytestmark = pytest.mark.gpu


def test_a_buffer_of_other_tokens():
    """The logits' buffer would be made anew under the bound router."""
    layer = RoutedExperts(64, 128, 8, 2)
    for x in (torch.zeros((9, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((3, 64), dtype=torch.bfloat16, device="cuda"),
              torch.zeros((4, 72), dtype=torch.bfloat16, device="cuda"), torch.zeros((4, 64), device="cuda"), torch.zeros((4, 64), dtype=torch.bfloat16),
              torch.zeros((1, 4, 64), dtype=torch.bfloat16, device="cuda")):
        with pytest.raises(FlexSpmvError, match="x "):
            DecodingStep(layer, 4, x=x)
    step = DecodingStep(layer, 4, x=torch.ones((4, 64), dtype=torch.bfloat16, device="cuda"))
    with torch.no_grad():
        assert torch.equal(step.launch(), layer(step.x))


def test_adapters_of_other_layers():
    stack = RoutedStack(64, 128, 8, 2, 2).eval()
    low = Adapter(torch.zeros((3, 8, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((3, 64, 8), dtype=torch.bfloat16, device="cuda"))
    for number in (1, 3):
        with pytest.raises(FlexSpmvError, match="2 layers"):
            DecodingStack(stack, 4, [low] * number)
    DecodingStack(stack, 4, [low] * 2).launch()
