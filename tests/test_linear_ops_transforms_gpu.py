"""The language-model operators under forward-mode differentiation and torch.jit.trace: refused, or recorded.  A
launch outside an autograd function would drop a tangent without a word and leave a trace an empty buffer."""
import pytest
import torch
from torch.autograd import forward_ad

from swiftx_b200.loss import linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _loss_operands(seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x, w = torch.randn(70, 24, generator=g, device=DEV), torch.randn(90, 24, generator=g, device=DEV)
    return x, w, torch.randint(0, 90, (70,), generator=g, device=DEV)


@pytest.mark.parametrize("which", [0, 1])
def test_loss_refuses_dual_numbers(which):
    x, w, y = _loss_operands()
    with forward_ad.dual_level():
        pair = [x, w]
        pair[which] = forward_ad.make_dual(pair[which], torch.ones_like(pair[which]))
        with pytest.raises(NotImplementedError):
            linear_cross_entropy(*pair, y)
        plain = linear_cross_entropy(x, w, y)          # no dual among the operands: the loss as ever
    assert torch.equal(plain, linear_cross_entropy(x, w, y))


def test_loss_is_a_node_of_a_trace():
    x, w, y = _loss_operands()
    f = torch.jit.trace(lambda x, w: linear_cross_entropy(x, w, y, reduction="none"), (x, w))
    x2, w2, _ = _loss_operands(1)
    assert torch.equal(f(x2, w2), linear_cross_entropy(x2, w2, y, reduction="none"))
