"""linear_log_probs and linear_distillation where a value is known far closer than the tolerances of a whole row: certain
words, small temperatures, logits that are exact.

Tolerances.  Exponents are (z - m) log2(e) / tau of logits z and their maximum m, so a row's largest term is 1 whatever the
temperature: the logarithm of the sum and the values are off by R = 2^-20 of 1 and the sizes of what is added (2^-21 for
exponentials, 2^-23 twice for an exponent, 2^-24 for each of the few terms that count), of the logits as they were summed.
"""
import math

import pytest
import torch

from swiftx_b200.log_probs import linear_log_probs
from swiftx_b200.loss import linear_distillation

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32
R = 2.0 ** -20
TEMPS = (1.0, 0.7, 1e-2, 1e-3, 1e-6, 1e-8, 1e-15)


def _certain(T, V, d, dtype, word, seed=0):
    """Rows whose softmax is all on one word.  A row's values add up to 5 to 60, its word's weights are 0.5 to 1.5 and all others' -90 to
    -30: with the operands' roundings (2^-8 each) the word's logit is at least 2.48 and the others' at most -148.8."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.rand(T, d, generator=g, device=DEV) + 0.5
    x *= torch.linspace(5, 60, T, device=DEV)[:, None] / x.sum(1, keepdim=True)
    w = -60 * (torch.rand(V, d, generator=g, device=DEV) + 0.5)
    w[word] = torch.rand(d, generator=g, device=DEV) + 0.5
    return x.to(dtype), w.to(dtype)


@pytest.mark.parametrize("T,V,d,dtype", [(40, 300, 64, BF), (300, 3001, 1024, BF), (8, 3001, 1024, BF), (3, 2500, 40, BF), (90, 700, 200, FP), (70, 2600, 1030, FP)])
@pytest.mark.parametrize("temp", TEMPS)
def test_a_certain_word(T, V, d, dtype, temp):
    """The others lie 151 / temperature or more below the word: 3001 e^-151 is below 2^-200, the log probability and the entropy are 0."""
    for word in (0, V // 2, V - 1):
        x, w = _certain(T, V, d, dtype, word, seed=V + word)
        y = torch.full((T,), word, device=DEV)
        out = linear_log_probs(x, w, y, top_k=min(5, V), temperature=temp)
        assert bool((out.top_ids[:, 0] == word).all())
        for t in (out.log_probs, -out.entropy, out.top_log_probs[:, 0]):
            assert bool((t <= 0).all()) and bool((t >= -R).all()), (float(t.max()), float(t.min()))
        assert bool((out.top_log_probs[:, 1:] <= -150).all())


@pytest.mark.parametrize("T,V,d,dtype", [(40, 300, 64, BF), (70, 3001, 256, BF), (3, 3001, 256, BF), (40, 300, 64, FP), (70, 3001, 1030, FP)])
@pytest.mark.parametrize("temp", [1e-3, 1e-4, 2.0 ** -16])
def test_small_differences_of_large_logits(T, V, d, dtype, temp):
    """Logits 32 + k 2^-16, exact in every sum, of a few words, all others far below: the distribution at a small temperature
    is that of the differences k 2^-16 / tau.  (The products' mean cut moves a difference by 2^-18 of itself at most.)"""
    g = torch.Generator(device=DEV).manual_seed(V)
    n = 24
    at = torch.randperm(V, generator=g, device=DEV)[:n]
    k = torch.arange(n, device=DEV) * max(1, int(temp * 2.0 ** 16 / 4))
    assert int(k[-1]) < 2 ** 12
    x = torch.zeros(T, d, device=DEV)
    x[:, 0], x[:, 1], x[:, 2] = 1, 1, 1
    w = torch.zeros(V, d, device=DEV)
    w[:, 0] = -64.0
    w[at, 0] = 32.0
    w[at, 1] = (k // 16).float() * 2.0 ** -12
    w[at, 2] = (k % 16).float() * 2.0 ** -16
    x, w = x.to(dtype), w.to(dtype)
    y = at[torch.arange(T, device=DEV) % n]
    l = torch.log_softmax((x.double() @ w.double().t()) / temp, 1)
    H = -(l.exp() * l).sum(1)
    out = linear_log_probs(x, w, y, top_k=n, temperature=temp)
    lp = l.gather(1, y[:, None])[:, 0]
    far = (R + 2.0 ** -18) * (l[:, at].abs().amax(1) + 1)
    for got, want in ((out.log_probs, lp), (out.entropy, H)):
        assert bool(((got.double() - want).abs() <= far).all()), float(((got.double() - want).abs() / far).max())
    assert torch.equal(out.top_ids[0], at.flip(0)) if int(k[1]) else True
    err = (out.top_log_probs.double() - l.gather(1, out.top_ids)).abs()
    assert bool((err <= far[:, None]).all()), float((err / far[:, None]).max())
    assert bool((out.log_probs <= 0).all()) and bool((out.top_log_probs <= 0).all()) and bool((out.entropy >= 0).all())


@pytest.mark.parametrize("dtype,T,V,d", [(BF, 600, 5001, 1024), (BF, 7, 5001, 1024), (FP, 200, 300, 256), (BF, 200, 900, 512)])
@pytest.mark.parametrize("temp", [1.0, 0.05])
def test_no_probability_is_above_one(dtype, T, V, d, temp):
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn(T, d, generator=g, device=DEV).to(dtype)
    w = (torch.randn(V, d, generator=g, device=DEV) * 12 / d ** 0.5).to(dtype)
    y = (x.double() @ w.double().t()).argmax(1)
    out = linear_log_probs(x, w, y, top_k=9, temperature=temp)
    assert bool((out.log_probs <= 0).all()) and bool((out.top_log_probs <= 0).all()) and bool((out.entropy >= 0).all())
    assert bool((out.top_log_probs[:, 1:] <= out.top_log_probs[:, :-1]).all())
    assert bool(torch.isfinite(torch.log1p(-torch.exp(out.top_log_probs[:, 5:].double()))).all())


@pytest.mark.parametrize("T,V,d,dtype", [(40, 300, 64, BF), (300, 3001, 1024, BF), (8, 3001, 1024, BF), (90, 700, 200, FP), (70, 2600, 1030, FP)])
@pytest.mark.parametrize("temp", (1.0, 1e-3, 1e-6, 1e-8, 1e-15))
def test_distillation_of_a_certain_word(T, V, d, dtype, temp):
    """Teacher and student are both certain of one word: no loss (R temperature^2), no gradient (temperature R of it)."""
    word = V - 2
    x, w = _certain(T, V, d, dtype, word, seed=V)
    x.requires_grad_(), w.requires_grad_()
    ids = torch.tensor([word, 5], device=DEV).expand(T, 2)
    logits = torch.tensor([0.0, -math.inf], device=DEV).expand(T, 2)
    loss = linear_distillation(x, w, ids, logits, temperature=temp)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert 0 <= float(loss.detach()) <= R * temp * temp
    assert float(dx.abs().max()) <= temp * R * float(w.detach().abs().max()) and float(dw.abs().max()) <= temp * R * float(x.detach().abs().max())


@pytest.mark.parametrize("T,V,top", [(20, 256, 6), (20, 300, 6), (5, 300, 0), (20, 3001, 6), (20, 3001, 0), (5, 3001, 6), (5, 3001, 0), (20, 3100, 40), (400, 2306, 100)])
def test_rows_without_a_word(T, V, top):
    """A row whose logits are all -inf gives NaN (as token_log_probs does) on any number of words and rows, its alternatives in order; the
    rows beside it stay as they were."""
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, 40, generator=g, device=DEV).to(BF)
    w = torch.randn(V, 40, generator=g, device=DEV).to(BF)
    y = torch.randint(0, V, (T,), generator=g, device=DEV)
    x[:, 0] = 0
    w[:, 0] = -3e38
    base = linear_log_probs(x, w, y, top_k=top)
    x[3, 0] = 3e38
    x.requires_grad_()
    out = linear_log_probs(x, w, y, top_k=top)
    rest = torch.arange(T, device=DEV) != 3
    for a, b in zip(out, base):
        if a is None:
            continue
        assert torch.equal(a[rest], b[rest])
        if a.is_floating_point():
            assert bool(torch.isnan(a[3]).all())
        else:
            assert torch.equal(a[3], torch.arange(top, device=DEV))
    dx, = torch.autograd.grad((out.log_probs + out.entropy).sum(), x)
    # (column 0 is a sum of -3e38 times the logits' gradients, whose magnitudes add up to as much as 2: over the largest fp32)
    assert bool(torch.isnan(dx[3]).all()) and bool(torch.isfinite(dx[rest][:, 1:]).all())
    loss = linear_distillation(x, w, y[:, None], torch.zeros(T, 1, device=DEV), reduction="none").detach()
    assert bool(torch.isnan(loss[3])) and bool(torch.isfinite(loss[rest]).all())


@pytest.mark.parametrize("T,V", [(20, 256), (20, 300), (20, 3001), (5, 3001)])
def test_logits_far_below_zero(T, V):
    """Logits of -1e24 and less, finite: the largest is certain, the others lie their distance below (each product rounded
    to 2^-22 of itself)."""
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.zeros(T, 16, device=DEV, dtype=BF)
    w = torch.zeros(V, 16, device=DEV, dtype=BF)
    x[:, 3] = 1e20
    w[:, 3] = -(torch.rand(V, generator=g, device=DEV) + 0.125) * 1e6
    z = x.double() @ w.double().t()
    y = z.argmax(1)
    out = linear_log_probs(x, w, y, top_k=8)
    ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :8]
    best = z.amax(1, keepdim=True)
    ties = (z == best).sum(1)
    assert torch.equal(out.top_ids, ids)
    for got in (out.log_probs + ties.log(), out.entropy - ties.log(), out.top_log_probs[:, 0] + ties.log()):
        assert bool((got.abs() <= R).all())
    far = z.gather(1, ids) - best
    assert bool(((out.top_log_probs - far).abs() <= 2.0 ** -20 * z.abs().amax() + R * far.abs() + 8).all())


@pytest.mark.parametrize("T,V,d,dtype", [(8, 3001, 1024, BF), (1, 5000, 2056, BF), (3, 2500, 40, BF), (9, 3001, 1024, BF), (300, 3001, 1024, BF), (8, 3001, 1024, FP)])
@pytest.mark.parametrize("temp", (1.0, 1e-2, 1e-3, 1e-6))
def test_gradients_of_a_certain_word(T, V, d, dtype, temp):
    """They vanish: dz is R / temperature of the upstream gradients at most."""
    x, w = _certain(T, V, d, dtype, 7, seed=T)
    x.requires_grad_(), w.requires_grad_()
    for top in (0, 4):
        out = linear_log_probs(x, w, torch.full((T,), 7, device=DEV), top_k=top, temperature=temp)
        for which in ((1.0, 0.0), (0.0, 1.0)):
            dx, dw = torch.autograd.grad(out[:2], (x, w), [torch.full((T,), c, device=DEV) for c in which], retain_graph=True)
            assert float(dx.abs().max()) <= R / temp * float(w.detach().abs().max()), (top, which, float(dx.abs().max()))
            assert float(dw.abs().max()) <= R / temp * float(x.detach().abs().sum(0).max()), (top, which, float(dw.abs().max()))


@pytest.mark.parametrize("T", [1, 5, 8])
@pytest.mark.parametrize("temp", [1.0, 0.02])
def test_few_rows_have_the_gradients_of_many(T, temp):
    """The first rows of a larger batch: the same logits, statistics and products with the weight, so the same gradient of x bit by bit."""
    g = torch.Generator(device=DEV).manual_seed(T)
    V, d = 3001, 520
    x = torch.randn(64, d, generator=g, device=DEV).to(BF)
    w = (torch.randn(V, d, generator=g, device=DEV) * 3 / d ** 0.5).to(BF)
    y = torch.randint(0, V, (64,), generator=g, device=DEV)
    a, b = torch.randn(64, generator=g, device=DEV), torch.randn(64, generator=g, device=DEV)
    got = []
    for n in (T, 64):
        xs = x[:n].clone().requires_grad_()
        out = linear_log_probs(xs, w, y[:n], temperature=temp)
        got.append(torch.autograd.grad(out[:2], xs, (a[:n], b[:n]))[0])
    assert torch.equal(got[0], got[1][:T])


@pytest.mark.parametrize("teacher", [FP, BF])
@pytest.mark.parametrize("temp", [1e-3, 0.5, 1.0, 3.0])
def test_teacher_logits_of_the_lowest_value(teacher, temp):
    """A teacher's softmax sees differences alone: entries that all stand at the type's lowest value (or at any other) are equal, and beside
    others they have no share."""
    g = torch.Generator(device=DEV).manual_seed(0)
    T, V, K = 30, 400, 5
    x, w = torch.randn(T, 24, generator=g, device=DEV), torch.randn(V, 24, generator=g, device=DEV)
    ids = torch.rand(T, V, generator=g, device=DEV).topk(K, 1).indices
    low = torch.finfo(teacher).min

    def run(logits):
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = linear_distillation(xs, ws, ids, logits.to(teacher), temperature=temp, reduction="none")
        return loss.detach(), *torch.autograd.grad(loss, (xs, ws), torch.ones_like(loss))
    zero = torch.zeros(T, K, device=DEV)
    equal = run(zero)
    assert all(bool(torch.isfinite(t).all()) for t in equal)
    for value in (low, -1e30, 3e38, -7.5):
        for a, b in zip(run(zero + value), equal):
            assert torch.equal(a, b)
    some = torch.arange(K, device=DEV) % 2 == 0
    # (unused words stand behind the others: a row's three terms are added in another order, 2^-23 of them, which are the loss and
    # the teacher's share of it, temperature^2 log 3)
    a, b = run(torch.where(some, zero, low)), run(torch.where(some, zero, -math.inf))
    assert bool(((a[0] - b[0]).abs() <= 2.0 ** -21 * (b[0].abs() + 2 * temp ** 2)).all())
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])


def _cut(d, dtype):
    """The share of a logit that the products' mean cut changes it by at most where its sum is exact: 0.25 2^-24 for each 16 of the terms that are
    summed in the tensor core at a time (8192; 512 of fp32 operands)."""
    return 0.25 * 2.0 ** -24 * min((d + 15) // 16, 512 if dtype == BF else 32)


@pytest.mark.parametrize("T,V,d,dtype", [(40, 300, 64, BF), (300, 3001, 1024, BF), (6, 3001, 1024, BF), (20, 400, 8192, BF), (20, 300, 16400, BF), (20, 300, 65536, BF),
                                         (60, 3001, 256, FP), (40, 300, 16384, FP)])
@pytest.mark.parametrize("kind", ["one word a row", "small integers"])
def test_exact_logits(T, V, d, dtype, kind):
    """Sums that no addition rounds: values are off by the mean cut of the logits' distances, and R."""
    g = torch.Generator(device=DEV).manual_seed(d)
    if kind == "one word a row":
        x = torch.zeros(T, d, device=DEV)
        at = torch.randint(0, d, (T,), generator=g, device=DEV)
        x[torch.arange(T, device=DEV), at] = 1.0
        w = torch.randn(V, d, generator=g, device=DEV).to(dtype) * 6
    else:
        x = torch.randint(-2, 3, (T, d), generator=g, device=DEV).float()
        w = torch.randint(-2, 3, (V, d), generator=g, device=DEV).to(dtype) * 2.0 ** -math.ceil(math.log2(d) / 2)
    x = x.to(dtype)
    y = torch.randint(0, V, (T,), generator=g, device=DEV)
    z = x.double() @ w.double().t()
    l = torch.log_softmax(z, 1)
    p = l.exp()
    H = -(p * l).sum(1)
    mean = (p * z).sum(1)
    out = linear_log_probs(x, w, y)
    lp, zy = l.gather(1, y[:, None])[:, 0], z.gather(1, y[:, None])[:, 0]
    for got, want, moved in ((out.log_probs, lp, (zy - mean).abs()), (out.entropy, H, (p * (z - mean[:, None]) ** 2).sum(1))):
        bound = _cut(d, dtype) * moved + R * (1 + lp.abs() + H)
        assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())
    loss = linear_distillation(x, w, y[:, None], torch.zeros(T, 1, device=DEV), reduction="none").double()
    bound = _cut(d, dtype) * (zy - mean).abs() + R * (1 + lp.abs() + H)
    assert bool(((loss + lp).abs() <= bound).all()), float(((loss + lp).abs() / bound).max())


@pytest.mark.parametrize("T,V,d,dtype", [(300, 2000, 1024, BF), (300, 2000, 4096, BF), (200, 600, 16384, BF), (200, 600, 65536, BF), (200, 600, 8200, BF),
                                         (300, 2000, 1024, FP), (100, 600, 16384, FP)])
def test_mean_error_of_dense_rows(T, V, d, dtype):
    """Terms of either sign are cut 0.20 to 0.27 2^-24 for each 16 of the n that come together, of which 0.23 are made up for: the entropy is off
    by 0.06 2^-24 n / 16 of the logits' variance on average over the rows (the roundings of each logit average out), and by 2^-22 of 1 and
    itself; distillation's loss by as much of its logits' distances.  Without the mean made up for they would be 4 times as far off."""
    g = torch.Generator(device=DEV).manual_seed(d)
    x = torch.randn(T, d, generator=g, device=DEV).to(dtype)
    w = (torch.randn(V, d, generator=g, device=DEV) * 2 / d ** 0.5).to(dtype)
    y = torch.randint(0, V, (T,), generator=g, device=DEV)
    z = x.double() @ w.double().t()
    l = torch.log_softmax(z, 1)
    p = l.exp()
    H = -(p * l).sum(1)
    mean = (p * z).sum(1)
    var = (p * (z - mean[:, None]) ** 2).sum(1)
    share = 0.06 / 0.25 * _cut(d, dtype)
    out = linear_log_probs(x, w, y)
    off = float((out.entropy.double() - H).mean().abs())
    assert off <= share * float(var.mean()) + 2.0 ** -22 * float(1 + H.mean()), (off, share * float(var.mean()))
    loss = linear_distillation(x, w, y[:, None], torch.zeros(T, 1, device=DEV))
    lp, zy = l.gather(1, y[:, None])[:, 0], z.gather(1, y[:, None])[:, 0]
    off = abs(float(loss) + float(lp.mean()))
    assert off <= share * float((zy - mean).mean().abs()) + 2.0 ** -22 * float(1 + lp.abs().mean()), (off, share)


def test_gradients_of_wide_bf16_rows():
    """9000 terms are summed in two pieces, forward and backward alike: a certain word's gradient vanishes, others are a logit's rounding
    (2^-8 of it) and the result's from float64 in the mean square."""
    T, V, d = 40, 300, 9000
    x, w = _certain(T, V, d, BF, 7)
    x.requires_grad_(), w.requires_grad_()
    out = linear_log_probs(x, w, torch.full((T,), 7, device=DEV), temperature=1e-3)
    for t, o in zip(torch.autograd.grad(out[:2], (x, w), [torch.ones(T, device=DEV)] * 2), (w, x)):
        assert float(t.abs().max()) <= 1e3 * R * T * float(o.detach().abs().max())
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(T, d, generator=g, device=DEV).to(BF).requires_grad_()
    w = (torch.randn(V, d, generator=g, device=DEV) * 2 / d ** 0.5).to(BF).requires_grad_()
    y = torch.randint(0, V, (T,), generator=g, device=DEV)
    got = torch.autograd.grad(linear_log_probs(x, w, y).log_probs.sum(), (x, w))
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    want = torch.autograd.grad(torch.log_softmax(xd @ wd.t(), 1).gather(1, y[:, None]).sum(), (xd, wd))
    for a, b in zip(got, want):
        assert float((a.double() - b).norm()) <= 2.0 ** -7 * float(b.norm())


@pytest.mark.parametrize("T,V,d,dtype,temp", [(300, 5001, 1024, BF, 1.0), (8, 5001, 1024, BF, 1.0), (1, 50001, 1024, BF, 1.0), (300, 300, 256, BF, 0.7), (200, 2000, 1024, FP, 1.0),
                                              (600, 5001, 2048, BF, 0.5)])
def test_values_in_the_mean_square(T, V, d, dtype, temp):
    """With n additions of a sum: the mean cut is made up for to 0.06 2^-24 n of a logit's distance from the mean logit, each logit is rounded by
    0.2 2^-24 n of the logits' standard deviation in the mean square (measured: 0.13 to 0.18), and a value by 2^-23 of 1 and itself."""
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, d, generator=g, device=DEV).to(dtype)
    w = (torch.randn(V, d, generator=g, device=DEV) * 2 / d ** 0.5).to(dtype)
    y = torch.randint(0, V, (T,), generator=g, device=DEV)
    z = x.double() @ w.double().t() / temp
    l = torch.log_softmax(z, 1)
    p = l.exp()
    H = -(p * l).sum(1)
    mean = (p * z).sum(1, keepdim=True)
    n = 4 * _cut(d, dtype)                                                # 2^-24 for each addition
    rms = lambda t: float(t.square().mean().sqrt())  # noqa: E731
    rounded = 0.2 * n * float(z.std()) * 2 ** 0.5
    out = linear_log_probs(x, w, y, top_k=20, temperature=temp)
    lp, zy = l.gather(1, y[:, None]), z.gather(1, y[:, None])
    bound = 0.06 * n * rms(zy - mean) + rounded + 2.0 ** -23 * rms(1 + lp.abs())
    assert rms(out.log_probs.double() - lp[:, 0]) <= bound
    ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :20]
    assert torch.equal(out.top_ids, ids)
    vals = l.gather(1, ids)
    bound = 0.06 * n * rms(z.gather(1, ids) - mean) + rounded + 2.0 ** -23 * rms(1 + vals.abs())
    assert rms(out.top_log_probs.double() - vals) <= bound
    var = (p * (z - mean).square()).sum(1)
    bound = 0.06 * n * rms(var) + rounded * rms((p * (l + H[:, None])).square().sum(1).sqrt()) + 2.0 ** -23 * rms(1 + H)
    assert rms(out.entropy.double() - H) <= bound
