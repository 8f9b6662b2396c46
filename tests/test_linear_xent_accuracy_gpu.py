"""linear_cross_entropy's fp32 products over wide operands: accuracy that does not fall with the width."""
import pytest
import torch
import torch.nn.functional as F

from swiftx_b200.loss import linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("T,V,d", [(64, 300, 4096), (33, 257, 16384), (300, 520, 1030)])
def test_fp32_logits_of_one_sign(T, V, d):
    """Operands of one sign, where what the tensor core cuts off each addition all goes the same way, and targets whose
    words are a tenth of the others', so that the loss is nine tenths of the largest logits.

    A logit is summed at most 512 terms at a time in the tensor core: 32 additions, at most 2^-23 each of the sum so far, which
    is half of the whole on average; those sums are added in fp32, 2^-24 each; the operands' pieces and the products left
    out take 8 2^-23 at most: e = (24 + d / 512) 2^-23 of the logit.  (d / 16 additions in one sum would cut off d / 16 times
    about 0.2 2^-23.)
    Statistics: 2^-20 of 1 + the logarithm of the sum of exponentials; the loss itself is rounded."""
    g = torch.Generator(device=DEV).manual_seed(d)
    x = 0.5 + torch.rand(T, d, generator=g, device=DEV)
    w = 0.5 + torch.rand(V, d, generator=g, device=DEV)
    w[: V // 2] *= 0.1
    y = torch.randint(0, V // 2, (T,), generator=g, device=DEV)
    got = linear_cross_entropy(x, w, y, reduction="none").double()
    logits = x.double() @ w.double().t()
    want = F.cross_entropy(logits, y, reduction="none")
    top = logits.amax(1)
    e = (24 + d / 512) * 2.0 ** -23 * top
    bound = 2 * e + 2.0 ** -20 * (1 + (torch.logsumexp(logits, 1) - top).abs()) + 2.0 ** -23 * want
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("T,V,d,reduction", [(130, 700, 1030, "mean"), (300, 300, 257, "none"), (70, 2100, 512, "sum"), (257, 90, 2049, "none"),
                                             (17900, 4200, 520, "mean")])        # two pieces of the vocabulary
def test_fp32_gradients_of_wide_operands(T, V, d, reduction):
    """A dlogit is off by its logit's error, e as above of |x_t| . |W_v|, with the statistics' 2^-20; dx and dW are sums
    of products of those, 256 terms at a time: less than (40 + n / 512) 2^-23 of the sum of magnitudes."""
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, d, generator=g, device=DEV)
    w = torch.randn(V, d, generator=g, device=DEV) * 2 / d ** 0.5
    y = torch.randint(0, V, (T,), generator=g, device=DEV)
    y[::7] = -100
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(xr, wr, y, reduction=reduction)
    c = torch.randn(loss.shape, generator=g, device=DEV)
    dx, dw = torch.autograd.grad(loss, (xr, wr), c)
    xd, wd = x.double(), w.double()
    logits = xd @ wd.t()
    live = y != -100
    rows = F.cross_entropy(logits, y, reduction="none")
    want = rows if reduction == "none" else rows.sum() / (live.sum() if reduction == "mean" else 1)
    e = (24 + d / 512) * 2.0 ** -23 * (xd.abs() @ wd.abs().t()).amax(1)
    assert bool(((loss.double() - want).abs() <= 2 * e.max() * (T if reduction == "sum" else 1) + 2.0 ** -18 * (1 + want.abs())).all())
    scale = torch.where(live, c.double().expand(T) / (live.sum() if reduction == "mean" else 1), torch.zeros(T, device=DEV, dtype=torch.float64))
    soft = torch.softmax(logits, 1)
    dl = soft * scale[:, None]
    dl[live, y[live]] -= scale[live]
    off = (2 * e + 2.0 ** -20)[:, None] * soft * scale[:, None].abs() + 2.0 ** -22 * dl.abs()
    for got, exact, mag, o, n in ((dx, dl @ wd, dl.abs() @ wd.abs(), off @ wd.abs(), V), (dw, dl.t() @ xd, dl.t().abs() @ xd.abs(), off.t() @ xd.abs(), T)):
        bound = o + (40 + n / 512) * 2.0 ** -23 * mag
        assert bool(((got.double() - exact).abs() <= bound + 1e-30).all()), float(((got.double() - exact).abs() / (bound + 1e-30)).max())
