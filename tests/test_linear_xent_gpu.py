"""linear_cross_entropy (swx_xent_fwd / _bwd) against float64 logits and torch's cross entropy on them.

Tolerances.  A logit is a sum of d products, 16 at a time in the tensor core (2^-23 of the sum of
magnitudes m_tv = |x_t| . |W_v| each time): e_t = (d / 16 + 8) 2^-23 max_v m_tv, and for fp32
operands (pieces to 2^-23) as much again.  With E = 2^-20 (two exponentials, the sum, the
logarithm):  |loss error| <= 2 e_t + E (1 + |lse_t|).  A dlogit's relative error is 2 e_t + E, and
one rounding to bf16 (2^-8) for bf16 operands; its product with W or x is a sum of n terms (2^-23 of
their magnitudes for each 16), and a bf16 result is rounded once more.
"""
import pytest
import torch
import torch.nn.functional as F

from swiftx_b200 import _lib
from swiftx_b200.loss import linear_cross_entropy
from swiftx_b200.sift import SiftConfig, SiftLM

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32


def _inputs(T, V, d, dtype, seed=0, ignored=0.1, ignore_index=-100):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, d, generator=g, device=DEV).to(dtype)
    w = (torch.randn(V, d, generator=g, device=DEV) * 2 / d ** 0.5).to(dtype)
    y = torch.randint(0, V, (T,), generator=g, device=DEV)
    drop = torch.rand(T, generator=g, device=DEV) < ignored
    return x, w, torch.where(drop, torch.full_like(y, ignore_index), y)


def _run(x, w, y, reduction="mean", dloss=None, ignore_index=-100):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(x, w, y, reduction=reduction, ignore_index=ignore_index)
    dloss = torch.ones_like(loss) if dloss is None else dloss
    dx, dw = torch.autograd.grad(loss, (x, w), dloss)
    assert _lib.load().swx_device_wait_status() == _lib.SWX_OK
    return loss.detach(), dx, dw


def _check(x, w, y, reduction, loss, dx, dw, dloss=None, ignore_index=-100):
    """dw may be fp32 for bf16 operands (an fp32 weight): rounded terms, a result that is not."""
    T, d = x.shape
    bf = x.dtype == BF
    xd, wd = x.double(), w.double()
    logits = xd @ wd.t()
    e = (d / 16 + 8) * 2.0 ** -23 * (xd.abs() @ wd.abs().t()).amax(1) * (1 if bf else 2)
    lse = torch.logsumexp(logits, 1)
    live = y != ignore_index
    rows = F.cross_entropy(logits, y, reduction="none", ignore_index=ignore_index)
    E = 2.0 ** -20
    row_bound = torch.where(live, 2 * e + E * (1 + lse.abs()), torch.zeros_like(e))
    if reduction == "none":
        want, bound, c = rows, row_bound, (torch.ones(T, device=DEV) if dloss is None else dloss).double()
    else:
        n = live.sum() if reduction == "mean" else 1
        want, bound = rows.sum() / n, row_bound.sum() / n + 2.0 ** -23 * (rows.sum() / n).abs()
        c = torch.full((T,), 1.0 if dloss is None else float(dloss), device=DEV, dtype=torch.float64) / n
    assert bool(((loss.double() - want).abs() <= bound).all()), float((loss.double() - want).abs().max())
    c = torch.where(live, c, torch.zeros_like(c))
    dl = torch.softmax(logits, 1)
    dl[live] -= F.one_hot(y[live], w.shape[0])
    dl *= c[:, None]
    # dlogit = (p - 1) c at the target: the error of p is relative to p, which is below 1 there
    mag = dl.abs()
    soft = torch.softmax(logits, 1) * c[:, None].abs()
    r = (2.0 ** -8 if bf else 2.0 ** -22)
    for got, other, m, s, n in ((dx, wd, mag, soft, w.shape[0]), (dw, xd, mag.t(), soft.t(), T)):
        want = (dl if got is dx else dl.t()) @ other
        u = (n / 16 + 16) * 2.0 ** -23
        ee = (2 * e + E)
        bound = (r + u) * (m @ other.abs()) + (((s * ee[:, None]) if got is dx else (s * ee[None])) @ other.abs())
        if got.dtype == BF:
            bound = bound + 2.0 ** -8 * want.abs()
        err = (got.double() - want).abs()
        assert bool((err <= 1.02 * bound + 1e-38).all()), f"largest error over bound {float((err / (1.02 * bound + 1e-38)).max()):.3g}"


@pytest.mark.parametrize("T,V,d,dtype,reduction", [
    (1, 1, 1, BF, "mean"), (1, 65, 17, BF, "sum"), (5, 300, 8, FP, "none"), (256, 256, 64, BF, "mean"),
    (257, 257, 65, BF, "none"), (300, 513, 200, FP, "mean"), (1000, 1003, 256, BF, "sum"), (33, 5001, 40, FP, "sum"),
    (130, 3001, 1030, BF, "mean"), (2048, 256, 256, BF, "mean"), (600, 2000, 100, FP, "none"),
])
def test_loss_and_gradients(T, V, d, dtype, reduction):
    x, w, y = _inputs(T, V, d, dtype, seed=T + V)
    y[0] = V - 1
    dloss = None
    if reduction == "none":
        dloss = torch.randn(T, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    _check(x, w, y, reduction, *_run(x, w, y, reduction, dloss), dloss)


def test_several_pieces_of_the_vocabulary():
    """More dlogit values than one piece holds: bf16 sums dx in fp32 between pieces; fp32 in dx itself."""
    for T, V, d, dtype in ((12288, 20000, 72, BF), (9000, 9001, 40, FP)):
        x, w, y = _inputs(T, V, d, dtype, seed=3)
        _check(x, w, y, "mean", *_run(x, w, y))


def test_reductions_weightings_and_scaled_gradients():
    x, w, y = _inputs(200, 777, 96, BF, seed=5)
    for red in ("mean", "sum"):
        dloss = torch.tensor(0.37, device=DEV)
        _check(x, w, y, red, *_run(x, w, y, red, dloss), dloss)


def test_ignored_tokens():
    x, w, y = _inputs(70, 200, 32, BF, ignored=0.0)
    # an index inside the vocabulary can be the ignored one
    y[::3] = 7
    _check(x, w, y, "mean", *_run(x, w, y, ignore_index=7), ignore_index=7)
    loss, dx, dw = _run(x, w, y, "none", ignore_index=7)
    assert torch.count_nonzero(loss[y == 7]) == 0 and torch.count_nonzero(dx[y == 7]) == 0
    none = torch.full_like(y, -100)
    loss, dx, dw = _run(x, w, none)
    assert torch.isnan(loss) and torch.count_nonzero(dx) == 0 and torch.count_nonzero(dw) == 0
    loss, dx, dw = _run(x, w, none, "sum")
    assert float(loss) == 0.0 and torch.count_nonzero(dx) == 0 and torch.count_nonzero(dw) == 0


def test_targets_outside_the_vocabulary_are_loud():
    x, w, y = _inputs(300, 500, 32, FP, ignored=0.0)
    for bad in (500, -1, 1 << 40):
        z = y.clone()
        z[4] = bad
        loss, dx, dw = _run(x, w, z, "none")
        assert torch.isnan(loss[4]) and torch.isnan(dx[4]).all() and torch.isfinite(loss[5:]).all() and torch.isfinite(dx[5:]).all()
        assert torch.isnan(_run(x, w, z)[0])


def test_infinite_and_extreme_logits():
    # a word masked out by weights of -inf (x > 0: its logits are -inf); fp32 operands have to be finite
    x, w, y = _inputs(40, 300, 32, BF, ignored=0.0)
    x = x.abs() + 0.125
    w[5] = -float("inf")
    y[y == 5] = 6
    loss, dx, dw = _run(x, w, y, "none")
    keep = torch.arange(300, device=DEV) != 5
    want, m = F.cross_entropy(x.double() @ w[keep].double().t(), y - (y > 5).long(), reduction="none"), x.double().abs() @ w[keep].double().abs().t()
    assert bool(((loss.double() - want).abs() <= 2 * 10 * 2.0 ** -23 * m.amax(1) + 2.0 ** -20 * (1 + want.abs())).all())
    assert torch.isnan(linear_cross_entropy(x.float(), w.float(), y))
    y[0] = 5                                            # and asked for: its loss is infinite
    assert torch.isinf(linear_cross_entropy(x, w, y, reduction="none")[0])
    x, w, y = _inputs(40, 300, 32, FP, ignored=0.0)
    big = linear_cross_entropy(x * 1e4, w, y, reduction="none")     # logits of 1e4: only their differences matter
    want = F.cross_entropy((x * 1e4).double() @ w.double().t(), y, reduction="none")
    m = ((x * 1e4).double().abs() @ w.double().abs().t()).amax(1)
    assert bool(((big.double() - want).abs() <= 2 * 2 * (2 + 8) * 2.0 ** -23 * m + 2.0 ** -20 * (1 + want.abs())).all())
    x[3, 2] = float("nan")
    assert torch.isnan(linear_cross_entropy(x, w, y, reduction="none")[3])


def test_layouts_and_partial_gradients():
    T, V, d = 160, 700, 64
    x, w, y = _inputs(T, V, d, BF, seed=8)
    base = _run(x, w, y)
    wide = torch.zeros(T, 2 * d, device=DEV, dtype=BF)
    wide[:, d:] = x
    odd_w = torch.zeros(V, d + 1, device=DEV, dtype=BF)
    odd_w[:, 1:] = w
    for xs, ws in ((wide[:, d:], w), (x, odd_w[:, 1:]), (x.t().contiguous().t(), w.t().contiguous().t())):
        for a, b in zip(base, _run(xs, ws, y)):
            assert torch.equal(a, b)
    shaped = linear_cross_entropy(x.view(4, 40, d), w, y.view(4, 40), reduction="none")
    assert shaped.shape == (4, 40)
    for want in ((True, False), (False, True)):
        xr, wr = x.detach().requires_grad_(want[0]), w.detach().requires_grad_(want[1])
        linear_cross_entropy(xr, wr, y).backward()
        got = (xr.grad, wr.grad)
        for g, b, on in zip(got, base[1:], want):
            assert (g is None) == (not on) and (g is None or torch.equal(g, b))
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, y), base[0])


@pytest.mark.parametrize("dtype", [BF, FP])
def test_single_rows_of_any_stride(dtype):
    """One token and one word, as views whose row stride is 0 or less than the row."""
    x, w, y = _inputs(1, 9, 24, dtype, ignored=0)
    base = _run(x, w, y)
    for stride in (0, 7):
        for a, b in zip(base, _run(x.as_strided((1, 24), (stride, 1)), w, y)):
            assert torch.equal(a, b)
    one = w[:1].as_strided((1, 24), (0, 1))
    loss, dx, dw = _run(x, one, torch.zeros_like(y))
    assert float(loss) == 0.0 and not dx.any() and not dw.any()


def test_fp32_weight_with_bf16_input_and_autocast():
    """The weight is rounded to bf16 for the products; its gradient comes back in fp32, not rounded again."""
    x, w, y = _inputs(260, 900, 80, FP, seed=4)
    x16 = x.to(BF)
    loss, dx, dw = _run(x16, w, y)
    assert dw.dtype == FP and dx.dtype == BF
    _check(x16, w.to(BF), y, "mean", loss, dx, dw)
    with torch.autocast("cuda", dtype=BF):
        a = _run(x, w, y)
    assert torch.equal(a[0], loss) and torch.equal(a[2], dw) and a[1].dtype == FP


def test_no_tokens():
    w = torch.randn(50, 16, device=DEV, requires_grad=True)
    x = torch.zeros(0, 16, device=DEV, requires_grad=True)
    y = torch.zeros(0, device=DEV, dtype=torch.int64)
    assert torch.isnan(linear_cross_entropy(x, w, y))
    linear_cross_entropy(x, w, y, reduction="sum").backward()
    assert torch.count_nonzero(w.grad) == 0 and x.grad.shape == (0, 16)
    assert linear_cross_entropy(x, w, y, reduction="none").shape == (0,)


def test_deterministic_streams_and_graphs():
    x, w, y = _inputs(1003, 3001, 72, BF, seed=6)
    a = _run(x, w, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _run(x, w, y)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    graphs = []
    for s in (6, 7):
        xs, ws, ys = _inputs(300, 2001, 72, BF, seed=s)
        xs.requires_grad_(), ws.requires_grad_()

        def f(xs=xs, ws=ws, ys=ys):
            loss = linear_cross_entropy(xs, ws, ys)
            return [loss.detach(), *torch.autograd.grad(loss, (xs, ws))]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = f()
        graphs.append((xs, f, g, r))
    for xs, *_ in graphs:
        with torch.no_grad():
            xs.mul_(0.5)
    for _, _, g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, f, _, r in graphs:
        for p, q in zip([t.clone() for t in r], f()):
            assert torch.equal(p, q)


def test_refusals():
    x, w, y = _inputs(10, 20, 16, BF)
    for args in ((x, w[:, :8], y), (x, w, y[:5]), (x, w, y.int()), (x.float(), w, y), (x.half(), w.half(), y), (x, w[0], y),
                 (x.double(), w.double(), y), (x[:, :0], w[:, :0], y)):
        with pytest.raises(ValueError):
            linear_cross_entropy(*args)
    with pytest.raises(ValueError):
        linear_cross_entropy(x, w, y, reduction="max")
    with pytest.raises(ValueError):
        linear_cross_entropy(x, w.float(), y, weight16=w[:5])
    with pytest.raises(RuntimeError):
        linear_cross_entropy(x.cpu(), w.cpu(), y.cpu())


@pytest.mark.parametrize("autocast", [False, True])
def test_language_model_loss(autocast):
    """SiftLM.loss against forward's own loss and gradients.  fp32: the head's two forms differ by
    their products' rounding (the library's fp32 products are off by d 2^-24 of their magnitudes, these by the
    bound above), which the backbone's gradients carry on: 2^-12 of each gradient's norm.  bf16: forward
    rounds the logits and their gradient to bf16 (2^-8 each) where loss() rounds the gradient once; a
    gradient is a sum of many such terms: 4 * 2^-8 of its norm."""
    torch.manual_seed(0)
    model = SiftLM(SiftConfig(vocab_size=300, d_model=64, n_layers=2)).to(DEV)
    idx = torch.randint(0, 300, (3, 50), device=DEV)
    tgt = torch.randint(0, 300, (3, 50), device=DEV)
    tgt[0, :7] = -100
    got = []
    for f in (lambda: model(idx, tgt)[1], lambda: model.loss(idx, tgt)):
        model.zero_grad()
        with torch.autocast("cuda", dtype=BF, enabled=autocast):
            loss = f()
        loss.backward()
        got.append((float(loss), {n: p.grad.clone() for n, p in model.named_parameters()}))
    tol = 4 * 2.0 ** -8 if autocast else 2.0 ** -12
    assert abs(got[0][0] - got[1][0]) <= tol * abs(got[0][0])
    for n, g in got[0][1].items():
        h = got[1][1][n]
        assert h.dtype == g.dtype and float((g - h).norm()) <= tol * float(g.norm()) + 1e-7, n


def test_attention_and_loss_train_together():
    """A layer of linear attention under the head's loss: a step's gradients against float64, and the same
    tokens through the recurrent step give the same hidden states."""
    from swiftx_b200.linear_attention import linear_attention, linear_attention_step
    torch.manual_seed(1)
    b, L, H, d, V = 2, 90, 2, 32, 500
    emb = (torch.randn(V, H * d, device=DEV) * 0.3).requires_grad_()
    proj = (torch.randn(3 * H * d, H * d, device=DEV) / (H * d) ** 0.5).requires_grad_()
    g = torch.tensor([-0.05, -0.5], device=DEV, requires_grad=True)
    idx = torch.randint(0, V, (b, L + 1), device=DEV)

    def hidden(emb, proj, g, attend):
        x = F.embedding(idx[:, :-1], emb)
        q, k, v = F.linear(x, proj).unflatten(-1, (3, H, d)).unbind(2)
        return x + attend(q, k, v, g).flatten(2)

    def slow(q, k, v, g):
        gap = torch.arange(L, device=DEV, dtype=q.dtype)
        m = torch.where(gap[:, None] >= gap[None], gap[:, None] - gap[None], torch.inf)
        w = torch.where(torch.isinf(m), 0.0, torch.exp(torch.where(torch.isinf(m), 0.0, m) * g[:, None, None]))
        return torch.einsum("bhts,bshd->bthd", torch.einsum("bthd,bshd->bhts", q, k) * d ** -0.5 * w, v)

    h = hidden(emb, proj, g, lambda q, k, v, g: linear_attention(q, k, v, g, scale=d ** -0.5))
    loss = linear_cross_entropy(h, emb, idx[:, 1:])
    grads = torch.autograd.grad(loss, (emb, proj, g))
    up = [t.detach().double().requires_grad_() for t in (emb, proj, g)]
    h64 = hidden(*up, slow)
    want = F.cross_entropy((h64 @ up[0].t()).flatten(0, 1), idx[:, 1:].flatten())
    gw = torch.autograd.grad(want, up)
    # fp32 throughout: every stage is good to (its additions) 2^-23 of its magnitudes, at most some
    # 2^-15 of each gradient's norm over the few stages here
    assert abs(float(loss) - float(want)) <= 2.0 ** -15 * float(want)
    for a, w in zip(grads, gw):
        assert float((a.double() - w).norm()) <= 2.0 ** -13 * float(w.norm())
    state = torch.zeros(b, H, d, d, device=DEV)
    with torch.no_grad():
        x = F.embedding(idx[:, :-1], emb)
        q, k, v = F.linear(x, proj).unflatten(-1, (3, H, d)).unbind(2)
        steps = [linear_attention_step(q[:, t], k[:, t], v[:, t], g.detach(), state, scale=d ** -0.5) for t in range(L)]
        again = x + torch.stack(steps, 1).flatten(2)
    assert float((again - h.detach()).norm()) <= 2.0 ** -15 * float(h.detach().norm())
