"""The language-model operators under forward-mode differentiation and torch.jit.trace: refused, or recorded.  A
launch outside an autograd function would drop a tangent without a word and leave a trace an empty buffer."""
import pytest
import torch
from torch.autograd import forward_ad

from swiftx_b200.linear_attention import linear_attention, linear_attention_step
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


def _attention_operands(seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q, k, v = (torch.randn(2, 100, 2, d, generator=g, device=DEV) for d in (24, 24, 40))
    return q, k, v, -torch.rand(2, 100, 2, generator=g, device=DEV), torch.randn(2, 2, 24, 40, generator=g, device=DEV)


@pytest.mark.parametrize("which", range(5))
def test_attention_refuses_dual_numbers(which):
    x = _attention_operands()
    with forward_ad.dual_level():
        dual = list(x)
        dual[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(NotImplementedError):
            linear_attention(*dual[:4], initial_state=dual[4])
        plain = linear_attention(*x[:4], initial_state=x[4])
    assert torch.equal(plain, linear_attention(*x[:4], initial_state=x[4]))


def test_attention_is_a_node_of_a_trace():
    def f(q, k, v, g, s0):
        return linear_attention(q, k, v, g, initial_state=s0, return_state=True)
    traced = torch.jit.trace(f, _attention_operands())
    x = _attention_operands(1)
    for a, b in zip(traced(*x), f(*x)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("which", range(5))
def test_step_refuses_dual_numbers(which):
    q, k, v, g, s = _attention_operands()
    x = [q[:, 0], k[:, 0], v[:, 0], g[:, 0], s]
    with forward_ad.dual_level(), torch.no_grad():
        dual = list(x)
        dual[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        before = s.clone()
        with pytest.raises(RuntimeError, match="not differentiable"):
            linear_attention_step(*dual)
        assert torch.equal(s, before)
        plain = linear_attention_step(*x)
    assert torch.equal(plain, linear_attention_step(*x[:4], before))


def test_step_refuses_a_trace():
    q, k, v, g, s = _attention_operands()
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda q, s: linear_attention_step(q, k[:, 0], v[:, 0], g[:, 0], s), (q[:, 0], s))
