"""linear_log_probs (swx_logprob_fwd / _bwd) and token_log_probs (swx_token_logprob) against float64.

Tolerances.  A logit is a sum of d products, 16 at a time in the tensor core (2^-23 of the sum of magnitudes
m_tv = |x_t| . |W_v| each time): e_t = (d / 16 + 8) 2^-23 max_v m_tv, and for fp32 operands (pieces to 2^-23) as much
again.  Statistics: sums of up to 128 terms one after the other (2^-24 each) and their joins, exponentials to 2^-21 and
the exponents' own rounding (2^-23 of the exponent): E = 2^-16 in all, of 1 and the sizes of what is added.  With the temperature tau
and the log probability l, the entropy H:
  l: 2 e / tau + E (1 + |l| + H);  H: its gradient's sum of magnitudes is at most 2 H / tau, so 2 H e / tau + E (1 + H).
Alternatives: the ids are those of the float64 logits (products of fp32 or bf16 values, summed in fp64 on both sides); values
as l.  dz = (g [v == y] - p (g + h (l + H))) / tau is off by p's relative error 2 e / tau + E on its part
and by h p times the errors of l and H; then one rounding to bf16 (2^-8 for bf16 operands, 2^-22 otherwise), the
products of n terms (2^-23 of their magnitudes for each 16), and a bf16 result's own rounding.
"""
import math

import pytest
import torch

from swiftx_b200 import _lib
from swiftx_b200.log_probs import LogProbs, linear_log_probs, token_log_probs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32
E = 2.0 ** -16


def _inputs(T, V, d, dtype, seed=0, ignored=0.1, std=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, d, generator=g, device=DEV).to(dtype)
    w = (torch.randn(V, d, generator=g, device=DEV) * std / d ** 0.5).to(dtype)
    y = torch.randint(0, V, (T,), generator=g, device=DEV)
    return x, w, torch.where(torch.rand(T, generator=g, device=DEV) < ignored, torch.full_like(y, -100), y)


def _order(z, k):
    """Ids of the k largest, the lowest first among equals."""
    return torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]


def _exact(z, y, temp, ignore=-100):
    """(log probabilities of every word, of y, entropy, live) of float64 logits."""
    l = torch.log_softmax(z / temp, 1)
    live = y != ignore
    lp = torch.where(live, l.gather(1, torch.where(live, y, 0)[:, None])[:, 0], 0.0)
    H = torch.where(live, -(l.exp() * torch.where(torch.isinf(l), 0.0, l)).sum(1), 0.0)
    return l, lp, H, live


def _errors(x, w, temp):
    e = (x.shape[1] / 16 + 8) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).amax(1)
    return e * (1 if x.dtype == BF else 2) / temp


def _within(got, want, bound, what):
    err = (got.double() - want).abs()
    assert bool((err <= bound + 1e-38).all()), f"{what}: largest error over bound {float((err / (bound + 1e-38)).max()):.3g}"


def _check_forward(out, x, w, y, temp, top, z=None, ignore=-100):
    z = x.double() @ w.double().t() if z is None else z
    e = _errors(x, w, temp)
    l, lp, H, live = _exact(z, y, temp, ignore)
    _within(out.log_probs, lp, torch.where(live, 2 * e + E * (1 + lp.abs() + H), 0.0), "log_probs")
    _within(out.entropy, H, torch.where(live, 2 * H * e + E * (1 + H), 0.0), "entropy")
    if not top:
        assert out.top_ids is None and out.top_log_probs is None
        return
    ids = torch.where(live[:, None], _order(z, top), -1)
    assert out.top_ids.dtype == torch.int64 and torch.equal(out.top_ids, ids)
    vals = torch.where(live[:, None], l.gather(1, ids.clamp(min=0)), 0.0)
    _within(out.top_log_probs, vals, torch.where(live[:, None], (2 * e + E * (1 + H))[:, None] + E * vals.abs(), 0.0), "top_log_probs")


def _check_gradients(x, w, y, temp, g, h, dx, dw, ignore=-100):
    z = x.double() @ w.double().t()
    e = _errors(x, w, temp)
    l, lp, H, live = _exact(z, y, temp, ignore)
    g, h = (torch.where(live, torch.zeros(x.shape[0], device=DEV, dtype=torch.float64) if t is None else t.double(), 0.0) for t in (g, h))
    p = l.exp()
    dz = -p * (g[:, None] + h[:, None] * (l + H[:, None]))
    off = dz.abs() * (2 * e + E)[:, None] + p * h.abs()[:, None] * ((2 * e + 2 * H * e + 2 * E * (1 + H))[:, None] + E * l.abs())
    dz[live, y[live]] += g[live]
    dz, off = dz / temp, off / temp + 2.0 ** -22 * g.abs()[:, None] * p / temp
    r = 2.0 ** -8 if x.dtype == BF else 2.0 ** -22
    for got, a, o, other, n in ((dx, dz, off, w.double(), w.shape[0]), (dw, dz.t(), off.t(), x.double(), x.shape[0])):
        if got is None:
            continue
        want = a @ other
        bound = ((r + (n / 16 + 16) * 2.0 ** -23) * a.abs() + 1.02 * o) @ other.abs()
        _within(got, want, 1.02 * bound + (2.0 ** -8 * want.abs() if got.dtype == BF else 0), "gradient")


def _upstream(T, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(T, generator=g, device=DEV), torch.randn(T, generator=g, device=DEV)


def _run(x, w, y, g, h, **kw):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    out = linear_log_probs(x, w, y, **kw)
    dx, dw = torch.autograd.grad(out[:2], (x, w), (g, h))
    assert _lib.load().swx_device_wait_status() == _lib.SWX_OK
    return LogProbs(*(t.detach() if t is not None else None for t in out)), dx, dw


@pytest.mark.parametrize("T,V,d,dtype,top,temp", [
    (1, 1, 1, BF, 1, 1.0), (1, 65, 17, BF, 65, 1.0), (5, 300, 8, FP, 20, 0.7), (256, 256, 64, BF, 0, 1.0), (257, 257, 65, BF, 7, 1.5),
    (300, 513, 200, FP, 0, 2.0), (70, 2049, 40, BF, 5, 1.0), (130, 3001, 72, FP, 128, 1.0), (33, 5001, 40, FP, 3, 0.5),
    (520, 9001, 264, BF, 31, 1.0), (64, 300, 1030, FP, 64, 1.0), (40, 20011, 128, BF, 128, 1.0), (3, 50001, 64, BF, 1, 3.0),
    (16, 9001, 1030, BF, 20, 1.0), (9, 4001, 33, BF, 0, 0.7), (1, 12345, 1024, BF, 128, 1.0), (8, 2049, 8, BF, 2, 1.0), (17, 2100, 64, BF, 4, 1.0),
    (15, 3001, 4104, BF, 11, 2.0), (2, 2500, 2304, BF, 5, 1.0), (7, 3001, 40, FP, 9, 1.0), (60, 4001, 1030, FP, 9, 1.0),
    (300, 9001, 520, BF, 100, 1.0), (2100, 5000, 2048, BF, 12, 1.0),
])
def test_values_alternatives_and_gradients(T, V, d, dtype, top, temp):
    x, w, y = _inputs(T, V, d, dtype, seed=T + V)
    y[0] = V - 1
    g, h = _upstream(T)
    out, dx, dw = _run(x, w, y, g, h, top_k=top, temperature=temp)
    _check_forward(out, x, w, y, temp, top)
    _check_gradients(x, w, y, temp, g, h, dx, dw)
    with torch.no_grad():
        for a, b in zip(linear_log_probs(x, w, y, top_k=top, temperature=temp), out):
            assert (a is None and b is None) or torch.equal(a, b)


def test_gradients_of_one_output_and_one_operand():
    T, V, d = 90, 700, 48
    x, w, y = _inputs(T, V, d, FP, seed=2)
    g, h = _upstream(T)
    for gg, hh in ((g, None), (None, h)):
        xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
        out = linear_log_probs(xr, wr, y)
        dx, dw = torch.autograd.grad((out.log_probs if hh is None else out.entropy,), (xr, wr), (gg if hh is None else hh,))
        _check_gradients(x, w, y, 1.0, gg, hh, dx, dw)
    for on in ((True, False), (False, True)):
        xr, wr = x.detach().requires_grad_(on[0]), w.detach().requires_grad_(on[1])
        out = linear_log_probs(xr, wr, y, top_k=2)
        assert not out.top_ids.requires_grad and not out.top_log_probs.requires_grad
        (out.log_probs.sum() + out.entropy.mean()).backward()             # upstream gradients that are broadcast
        _check_gradients(x, w, y, 1.0, torch.ones(T, device=DEV), torch.full((T,), 1 / T, device=DEV), xr.grad, wr.grad)
        assert (xr.grad is not None, wr.grad is not None) == on


def test_gradients_against_differences():
    """sum(g l + h H) along a direction: the operator's own central difference is off by its values' errors over the
    step, and from the derivative by what float64 says the step makes."""
    T, V, d, temp = 40, 333, 24, 0.8
    x, w, y = _inputs(T, V, d, FP, seed=3)
    g, h = _upstream(T)
    u, v = torch.randn_like(x) / 8, torch.randn_like(w) / 8
    _, dx, dw = _run(x, w, y, g, h, temperature=temp)
    got = float((dx.double() * u).sum() + (dw.double() * v).sum())
    step = 2.0 ** -4

    def f64(t):
        _, lp, H, _ = _exact((x + t * u).double() @ (w + t * v).double().t(), y, temp)
        return float((g * lp + h * H).sum())

    def f(t):
        out = linear_log_probs(x + t * u, w + t * v, y, temperature=temp)
        return float((g.double() * out.log_probs + h * out.entropy).sum())
    diff, diff64 = (f(step) - f(-step)) / (2 * step), (f64(step) - f64(-step)) / (2 * step)
    xd, wd = x.double().requires_grad_(), w.double().requires_grad_()
    _, lp, H, _ = _exact(xd @ wd.t(), y, temp)
    gx, gw = torch.autograd.grad((g * lp + h * H).sum(), (xd, wd))
    exact = float((gx * u).sum() + (gw * v).sum())
    _, lp, H, _ = _exact(x.double() @ w.double().t(), y, temp)
    e = 1.5 * _errors(x, w, temp)                                         # the moved operands are a little larger
    noise = float((g.abs() * (2 * e + E * (2 + 2 * lp.abs() + 2 * H)) + h.abs() * (3 * H * e + E * (2 + 2 * H))).sum())
    assert abs(diff - diff64) <= noise / step
    assert abs(got - diff) <= abs(exact - diff64) + noise / step + 2.0 ** -12 * float((gx * u).abs().sum() + (gw * v).abs().sum())


@pytest.mark.parametrize("dtype,V", [(BF, 300), (BF, 7001), (FP, 300), (FP, 7001)])
def test_equal_logits_go_to_the_lowest_word(dtype, V):
    """Words with the same weights, in one group of 32 columns and far apart; rows of zeros, where all words are equal."""
    T, d, top = 70, 40, 40
    x, w, y = _inputs(T, V, d, dtype, seed=4, ignored=0)
    source = torch.arange(V, device=DEV)
    source[V // 2:] = torch.arange(V - V // 2, device=DEV)                # the second half repeats the first
    source[5:9] = 4
    source[V - 3:] = 4
    x[7], x[8] = 0, -x[9]
    first, back = torch.unique(source, return_inverse=True)
    z = (x.double() @ w[first].double().t())[:, back]                     # equal words have equal logits here too
    w = w[source].contiguous()
    out = linear_log_probs(x, w, y, top_k=top)
    _check_forward(out, x, w, y, 1.0, top, z=z)
    assert torch.equal(out.top_ids[7], torch.arange(top, device=DEV))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_large_logits_gathered_in_few_groups(dtype):
    """Groups of 32 words go round 128 threads: the largest logits all in the groups of four of them; rows of a few values."""
    T, V, d = 4, 100000, 8
    x, w, y = _inputs(T, V, d, dtype, seed=13, ignored=0)
    group = torch.arange(V, device=DEV) // 32
    x[:, 0] = 1.0
    w[:, 0] = torch.where(group % 128 < 4, 40.0, 0.0)
    w[:, 1] = 0
    for top in (1, 3, 60, 128):
        _check_forward(linear_log_probs(x, w, y, top_k=top), x, w, y, 1.0, top)
    x[1:] = 0
    x[1:, 0] = 1.0                                                        # 12512 words alike
    _check_forward(linear_log_probs(x, w, y, top_k=9), x, w, y, 1.0, 9)


def test_close_logits_are_ordered_exactly():
    """Words whose logits differ by a 2^-26th, far below what an fp32 sum tells apart."""
    d, V, top = 64, 4001, 24
    x = torch.ones(3, d, device=DEV)
    w = torch.zeros(V, d, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    at = torch.randperm(V, generator=g, device=DEV)[:24]
    w[:, 0] = -1.0
    w[at, 0] = 8.0
    w[at, 1] = 2.0 ** -23 * torch.arange(24, device=DEV)
    out = linear_log_probs(x, w, torch.zeros(3, dtype=torch.int64, device=DEV), top_k=top)
    assert torch.equal(out.top_ids, at.flip(0).expand(3, top))


def test_ignored_and_bad_targets():
    x, w, y = _inputs(70, 200, 32, BF, ignored=0.0)
    y[::3] = 7                                                            # an index inside the vocabulary can be the ignored one
    g, h = _upstream(70)
    out, dx, dw = _run(x, w, y, g, h, top_k=4, ignore_index=7)
    _check_forward(out, x, w, y, 1.0, 4, ignore=7)
    _check_gradients(x, w, y, 1.0, g, h, dx, dw, ignore=7)
    assert not dx[y == 7].any() and bool((out.top_ids[y == 7] == -1).all())
    none = torch.full_like(y, -100)
    out, dx, dw = _run(x, w, none, g, h, top_k=4)
    assert not any(t.any() for t in (*out[:3], dx, dw)) and bool((out.top_ids == -1).all())
    base, bdx, _ = _run(x, w, y, g, h)
    for bad in (200, -1, 1 << 40):
        b = y.clone()
        b[4] = bad
        out, dx, dw = _run(x, w, b, g, h)
        assert torch.isnan(out.log_probs[4]) and torch.isnan(dx[4]).all()
        assert torch.equal(out.log_probs[5:], base.log_probs[5:]) and torch.equal(dx[5:], bdx[5:])


@pytest.mark.parametrize("T,V", [(40, 300), (40, 3000), (11, 3000)])
def test_words_that_weights_of_infinity_mask(T, V):
    x, w, y = _inputs(T, V, 32, BF, ignored=0.0)
    x = x.abs() + 0.125
    keep = torch.ones(V, dtype=torch.bool, device=DEV)
    keep[[5, 40, 41, V - 1]] = False
    keep[96:160] = False                                                  # whole groups
    w[~keep] = -math.inf
    y[~keep[y]] = 6
    out = linear_log_probs(x, w, y, top_k=20)
    to = torch.cumsum(keep, 0) - 1
    kept = torch.nonzero(keep)[:, 0]
    want = linear_log_probs(x, w[kept].contiguous(), to[y], top_k=20)
    # the same words, summed in other groups: twice E
    for a, b in zip(out[:3], want[:3]):
        assert bool(((a - b).abs() <= 2 * E * (4 + b.abs())).all())
    assert torch.equal(out.top_ids, kept[want.top_ids])
    y[0] = 5
    assert float(linear_log_probs(x, w, y).log_probs[0]) == -math.inf
    x[3, 2] = math.nan
    out = linear_log_probs(x, w, y, top_k=20)
    assert torch.isnan(out.log_probs[3]) and torch.isnan(out.entropy[3])
    assert bool((out.top_ids >= 0).all() & (out.top_ids < V).all()) and out.top_ids[3].unique().numel() == 20


def test_layouts():
    T, V, d = 160, 2700, 64
    x, w, y = _inputs(T, V, d, BF, seed=8)
    g, h = _upstream(T)
    base = _run(x, w, y, g, h, top_k=9)
    wide = torch.zeros(T, 2 * d, device=DEV, dtype=BF)
    wide[:, d:] = x
    odd_w = torch.zeros(V, d + 1, device=DEV, dtype=BF)
    odd_w[:, 1:] = w
    for xs, ws in ((wide[:, d:], w), (x, odd_w[:, 1:]), (x.t().contiguous().t(), w.t().contiguous().t())):
        for a, b in zip((*base[0], *base[1:]), (lambda r: (*r[0], *r[1:]))(_run(xs, ws, y, g, h, top_k=9))):
            assert torch.equal(a, b)
    shaped = linear_log_probs(x.view(4, 40, d), w, y.view(4, 40), top_k=9)
    assert shaped.log_probs.shape == shaped.entropy.shape == (4, 40) and shaped.top_ids.shape == shaped.top_log_probs.shape == (4, 40, 9)
    for a, b in zip(shaped, base[0]):
        assert torch.equal(a.reshape(b.shape), b)
    xf, wf, y = _inputs(T, V, d, FP, seed=9)
    base = linear_log_probs(xf, wf, y, top_k=9)
    odd = torch.zeros(V, d + 1, device=DEV)
    odd[:, 1:] = wf
    again = linear_log_probs(xf, odd[:, 1:], y, top_k=9)
    assert torch.equal(base.top_ids, again.top_ids) and torch.equal(base.log_probs, again.log_probs)
    one = linear_log_probs(xf[:1].as_strided((1, d), (0, 1)), wf, y[:1], top_k=9)
    assert torch.equal(one.top_ids, base.top_ids[:1])


def test_fp32_weight_with_bf16_input_and_autocast():
    x, w, y = _inputs(260, 900, 80, FP, seed=4)
    x16 = x.to(BF)
    g, h = _upstream(260)
    out, dx, dw = _run(x16, w, y, g, h, top_k=6)
    assert dw.dtype == FP and dx.dtype == BF
    _check_forward(out, x16, w.to(BF), y, 1.0, 6)
    _check_gradients(x16, w.to(BF), y, 1.0, g, h, dx, dw)
    with torch.autocast("cuda", dtype=BF):
        a, _, dw2 = _run(x, w, y, g, h, top_k=6)
    assert all(torch.equal(p, q) for p, q in zip(a, out)) and torch.equal(dw, dw2)
    b = linear_log_probs(x16, w, y, top_k=6, weight16=w.to(BF))
    assert all(torch.equal(p, q) for p, q in zip(b, out))


def test_no_tokens():
    w = torch.randn(50, 16, device=DEV, requires_grad=True)
    x = torch.zeros(0, 16, device=DEV, requires_grad=True)
    out = linear_log_probs(x, w, torch.zeros(0, device=DEV, dtype=torch.int64), top_k=3)
    assert out.log_probs.shape == (0,) and out.top_ids.shape == (0, 3)
    (out.log_probs.sum() + out.entropy.sum()).backward()
    assert not w.grad.any() and x.grad.shape == (0, 16)
    assert token_log_probs(torch.zeros(0, 9, device=DEV), top_k=2).top_ids.shape == (0, 2)


def test_several_pieces_of_the_vocabulary():
    T, V, d = 12288, 20000, 72
    x, w, y = _inputs(T, V, d, BF, seed=3)
    g, h = _upstream(T)
    out, dx, dw = _run(x, w, y, g, h)
    _check_gradients(x, w, y, 1.0, g, h, dx, dw)


@pytest.mark.parametrize("T,V,d,dtype,top", [(8700, 3001, 40, BF, 6), (8193, 300, 24, FP, 3), (16400, 2500, 32, FP, 9), (9000, 700, 33, BF, 0)])
def test_more_rows_than_one_product_takes(T, V, d, dtype, top):
    x, w, y = _inputs(T, V, d, dtype, seed=14)
    out = linear_log_probs(x, w, y, top_k=top)
    _check_forward(out, x, w, y, 1.0, top)
    xo = torch.zeros(T, d + 3, device=DEV, dtype=dtype)[:, 3:]            # rows off 16 bytes
    xo.copy_(x)
    for a, b in zip(linear_log_probs(xo, w, y, top_k=top), out):
        assert (a is None and b is None) or torch.equal(a, b) or (a.is_floating_point() and float((a - b).abs().max()) <= E)


@pytest.mark.parametrize("T,V,d,dtype,top", [(4001, 10007, 201, FP, 20), (2600, 6001, 521, BF, 40), (2200, 1024, 1024, BF, 12)])
def test_norms_of_the_words(T, V, d, dtype, top):
    """Sizes whose candidates' bound comes from the longest word, here the last one: eager, and replayed with other operands."""
    assert T * (top + 4) > V and T * (top + 4) * d * (4 if dtype == FP else 2) > 64 << 20 and V * d < 32 << 20
    x, w, y = _inputs(T, V, d, dtype, seed=T)
    w[-1] *= 2
    with torch.no_grad():
        _check_forward(linear_log_probs(x, w, y, top_k=top), x, w, y, 1.0, top)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = linear_log_probs(x, w, y, top_k=top)
        w.mul_(-2), x.mul_(0.5)
        graph.replay()
        _check_forward(out, x, w, y, 1.0, top)
        for a, b in zip(out, linear_log_probs(x, w, y, top_k=top)):
            assert torch.equal(a, b)
    assert _lib.load().swx_device_wait_status() == _lib.SWX_OK


def test_deterministic_streams_and_graphs():
    x, w, y = _inputs(603, 5001, 72, BF, seed=6)
    g, h = _upstream(603)
    a = _run(x, w, y, g, h, top_k=11)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _run(x, w, y, g, h, top_k=11)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for p, q in zip((*a[0], *a[1:]), (*b[0], *b[1:])):
        assert torch.equal(p, q)
    graphs = []
    for s in (6, 7):
        xs, ws, ys = _inputs(300, 4001, 72, BF, seed=s)
        zs = torch.randn(5, 4001, device=DEV)
        xs.requires_grad_(), ws.requires_grad_()

        def f(xs=xs, ws=ws, ys=ys, zs=zs):
            out = linear_log_probs(xs, ws, ys, top_k=5)
            more = token_log_probs(zs, ys[:5], top_k=5)
            return [t.detach() for t in (*out, *more)] + list(torch.autograd.grad(out[:2], (xs, ws), (g[:300], h[:300])))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = f()
        graphs.append((xs, zs, f, graph, r))
    for xs, zs, *_ in graphs:
        with torch.no_grad():
            xs.mul_(0.5), zs.mul_(2)
    for _, _, _, graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, _, f, _, r in graphs:
        for p, q in zip([t.clone() for t in r], f()):
            assert torch.equal(p, q)


# ------------------------------------------------------------------ from logits
def _check_tokens(z, y, top, temp, out, ignore=-100):
    """Sums of up to V / 256 terms of a thread and their joins, exponents rounded to 2^-23 of them."""
    zd = z.double()
    e = (z.shape[1] / 256 + 64) * 2.0 ** -24
    target = torch.zeros(z.shape[0], dtype=torch.int64, device=DEV) if y is None else y
    l, lp, H, live = _exact(zd, target, temp, ignore)
    if y is None:
        assert out.log_probs is None
    else:
        fin = torch.isfinite(lp)
        assert torch.equal(out.log_probs[~fin].double(), lp[~fin])
        _within(out.log_probs[fin], lp[fin], torch.where(live, (e + 2.0 ** -21) * (1 + lp.abs() + H), 0.0)[fin], "log_probs")
    _within(out.entropy, H, torch.where(live, (2 * e + 2.0 ** -20) * (1 + H), 0.0), "entropy")
    if top:
        ids = torch.where(live[:, None], _order(zd, top), -1)
        assert torch.equal(out.top_ids, ids)
        vals = torch.where(live[:, None], l.gather(1, ids.clamp(min=0)), 0.0)
        fin = torch.isfinite(vals)
        assert torch.equal(fin, torch.isfinite(out.top_log_probs))
        bound = (e + 2.0 ** -21) * (1 + H[:, None] + torch.where(fin, vals.abs(), 0.0))
        _within(torch.where(fin, out.top_log_probs, 0.0), torch.where(fin, vals, 0.0), torch.where(live[:, None], bound, 0.0), "top_log_probs")


@pytest.mark.parametrize("R,V,dtype,top,temp", [
    (1, 1, FP, 1, 1.0), (3, 7, BF, 7, 1.0), (1, 256, FP, 5, 1.0), (19, 10007, BF, 8, 0.7), (700, 65, FP, 65, 1.0), (2, 50001, FP, 128, 2.0),
    (300, 8191, BF, 0, 1.0), (40, 32768, BF, 20, 1.0), (1, 262147, FP, 64, 1.0), (4, 131, FP, 128, 1.0), (600, 4096, FP, 1, 1.0),
])
def test_tokens(R, V, dtype, top, temp):
    g = torch.Generator(device=DEV).manual_seed(R + V)
    z = (torch.randn(R, V, generator=g, device=DEV) * 3).to(dtype)
    y = torch.randint(0, V, (R,), generator=g, device=DEV)
    _check_tokens(z, y, top, temp, token_log_probs(z, y, top_k=top, temperature=temp))
    _check_tokens(z, None, top, temp, token_log_probs(z, top_k=top, temperature=temp))


def test_tokens_in_hard_orders():
    """Rows in rising and falling order, constant ones, few distinct values: what the running threshold meets at worst."""
    V, top = 40000, 100
    up = torch.arange(V, device=DEV, dtype=FP) / 256
    rows = torch.stack([up, up.flip(0), torch.zeros(V, device=DEV), (torch.arange(V, device=DEV) % 3).float(), torch.full((V,), -1e30, device=DEV),
                        torch.where(torch.arange(V, device=DEV) < V - 50, 0.0, 1.0), -torch.zeros(V, device=DEV)])
    rows[6, ::2] = 0.0                                                    # zeros of either sign are equal
    y = torch.arange(7, device=DEV)
    # large values in the shares of few threads (16-byte pieces go round 256 threads), in falling and rising order
    heavy = torch.where(torch.arange(V, device=DEV) // 4 % 256 < 10, 1000 + up, up)
    rows = torch.cat([rows, heavy[None], (heavy.max() - heavy)[None], torch.where(heavy > 1000, 5.0, up)[None]])
    y = torch.arange(10, device=DEV)
    for n in (V, V - 1, 9000):
        z = rows[:, :n]
        _check_tokens(z, y, top, 1.0, token_log_probs(z, y, top_k=top))
    many = rows.repeat(60, 1)                                             # one CTA for each row
    _check_tokens(many, y.repeat(60), top, 1.0, token_log_probs(many, y.repeat(60), top_k=top))
    _check_tokens(rows[:, :2048], y, 64, 1.0, token_log_probs(rows[:, :2048], y, top_k=64))        # the smaller CTAs
    _check_tokens(rows[:, :2047], y, 2, 1.0, token_log_probs(rows[:, :2047], y, top_k=2))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_tokens_masked(dtype):
    g = torch.Generator(device=DEV).manual_seed(5)
    V, top = 6007, 12
    z = torch.randn(9, V, generator=g, device=DEV).to(dtype)
    y = torch.zeros(9, dtype=torch.int64, device=DEV)
    z[:, 5:] = torch.where(torch.rand(9, V - 5, generator=g, device=DEV) < 0.9, torch.tensor(-math.inf, device=DEV, dtype=dtype), z[:, 5:])
    z[1, 1:] = -math.inf                                                  # one word left
    z[2, 4:] = -math.inf                                                  # fewer than the alternatives
    z[7, 1:] = torch.finfo(dtype).min                                     # the type's lowest value as a mask
    z[8] = torch.finfo(dtype).min                                         # and in every place: all words alike
    _check_tokens(z, y, top, 1.0, token_log_probs(z, y, top_k=top))
    _check_tokens(z[:7], y[:7], top, 0.5, token_log_probs(z[:7], y[:7], top_k=top, temperature=0.5))
    assert float(token_log_probs(z, y).entropy[1]) == 0.0 and float(token_log_probs(z, y).log_probs[1]) == 0.0
    y[1] = 3
    assert float(token_log_probs(z, y).log_probs[1]) == -math.inf         # a word that is not allowed
    # nothing left, a NaN, an infinity: NaN values, ids in order, the other rows as they were
    base = token_log_probs(z, y, top_k=top)
    z[4] = -math.inf
    z[5, 77] = math.nan
    z[6, 99] = math.inf
    out = token_log_probs(z, y, top_k=top)
    for r in (4, 5, 6):
        assert torch.isnan(out.log_probs[r]) and torch.isnan(out.entropy[r]) and torch.isnan(out.top_log_probs[r]).all()
    assert torch.equal(out.top_ids[4], torch.arange(top, device=DEV)) and int(out.top_ids[6, 0]) == 99 and int(out.top_ids[5, 0]) == 77
    for a, b in zip(out, base):
        assert torch.equal(a[[0, 1, 2, 3, 7, 8]], b[[0, 1, 2, 3, 7, 8]])


def test_tokens_ignored_and_layouts():
    g = torch.Generator(device=DEV).manual_seed(6)
    wide = torch.randn(12, 2 * 5003, generator=g, device=DEV)
    y = torch.randint(0, 5003, (12,), generator=g, device=DEV)
    y[3] = -100
    for z in (wide[:, :5003], wide[:, 5001:10004], wide.to(BF)[:, 3:5006], wide[:, :5003].t().contiguous().t(), wide[:1, :5003].expand(12, 5003)):
        out = token_log_probs(z, y, top_k=6)
        _check_tokens(z, y, 6, 1.0, out)
        assert float(out.log_probs[3]) == float(out.entropy[3]) == 0.0 and bool((out.top_ids[3] == -1).all())
    z = wide[:, :5003]
    for bad in (5003, -1, 1 << 40):
        b = y.clone()
        b[5] = bad
        assert torch.isnan(token_log_probs(z, b).log_probs[5])
    shaped = token_log_probs(z.reshape(3, 4, 5003), y.view(3, 4), top_k=6)
    flat = token_log_probs(z, y, top_k=6)
    assert shaped.entropy.shape == (3, 4) and torch.equal(shaped.top_ids.view(12, 6), flat.top_ids)
    one = token_log_probs(z[0], y[0], top_k=6)
    assert one.log_probs.shape == () and one.top_ids.shape == (6,) and torch.equal(one.top_ids, flat.top_ids[0])


def test_both_forms_agree():
    """The scoring of hidden states and of the logits that a library product makes of them: ids up to logits that
    rounding brings closer than both sides' errors, values to those errors."""
    x, w, y = _inputs(200, 3001, 64, FP, seed=11, ignored=0)
    a = linear_log_probs(x, w, y, top_k=10)
    b = token_log_probs(x @ w.t(), y, top_k=10)
    e = _errors(x, w, 1.0) + 64 * 2.0 ** -24 * (x.abs() @ w.abs().t()).amax(1)
    bound = 4 * e + 2 * E * (1 + a.log_probs.abs() + a.entropy)
    for p, q in zip(a[:2], b[:2]):
        _within(p, q.double(), bound, "forms")
    _within(a.top_log_probs, b.top_log_probs.double(), (4 * e + 2 * E * (1 + a.entropy))[:, None] + 2 * E * a.top_log_probs.abs(), "forms")


def test_refusals():
    x, w, y = _inputs(10, 20, 16, BF)
    for args in ((x, w[:, :8], y), (x, w, y[:5]), (x, w, y.int()), (x.float(), w, y), (x.half(), w.half(), y), (x, w[0], y),
                 (x.double(), w.double(), y), (x[:, :0], w[:, :0], y)):
        with pytest.raises(ValueError):
            linear_log_probs(*args)
    for kw in (dict(top_k=21), dict(top_k=-1), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf),
               dict(weight16=w[:5])):
        with pytest.raises(ValueError):
            linear_log_probs(x, w.float() if "weight16" in kw else w, y, **kw)
    with pytest.raises(ValueError):
        linear_log_probs(x, w.repeat(10, 1), y, top_k=129)
    z = torch.randn(10, 20, device=DEV)
    for args, kw in (((z.double(),), {}), ((z, y.int()), {}), ((z, y[:4]), {}), ((z[:, :0],), {}), ((z,), dict(top_k=21)), ((z,), dict(temperature=0))):
        with pytest.raises(ValueError):
            token_log_probs(*args, **kw)
    with pytest.raises(RuntimeError, match="not differentiable"):
        token_log_probs(z.clone().requires_grad_())
    with torch.no_grad():
        token_log_probs(z.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: token_log_probs(t).entropy, (z,))
    with pytest.raises(RuntimeError):
        token_log_probs(z.cpu())
    with pytest.raises(RuntimeError):
        linear_log_probs(x.cpu(), w.cpu(), y.cpu())


def test_transforms():
    from torch.autograd import forward_ad
    x, w, y = _inputs(50, 90, 24, FP)
    with forward_ad.dual_level():
        for which in (0, 1):
            pair = [x, w]
            pair[which] = forward_ad.make_dual(pair[which], torch.ones_like(pair[which]))
            with pytest.raises(NotImplementedError):
                linear_log_probs(*pair, y)
        with pytest.raises(RuntimeError, match="not differentiable"):
            token_log_probs(forward_ad.make_dual(x, torch.ones_like(x)))
        plain = linear_log_probs(x, w, y, top_k=3)
    for a, b in zip(plain, linear_log_probs(x, w, y, top_k=3)):
        assert torch.equal(a, b)
    f = torch.jit.trace(lambda x, w: tuple(linear_log_probs(x, w, y, top_k=3)), (x, w))
    x2, w2, _ = _inputs(50, 90, 24, FP, seed=1)
    for a, b in zip(f(x2, w2), linear_log_probs(x2, w2, y, top_k=3)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,V,d,dtype,top", [(8700, 6001, 521, BF, 40), (16500, 4500, 264, FP, 9)])
def test_norms_of_the_words_over_several_products(T, V, d, dtype, top):
    """A teacher's batch: the bound of the candidates comes from the longest word, here the last one, read once for all rows."""
    assert T > 8192 and T * (top + 4) > V and T * (top + 4) * d * (4 if dtype == FP else 2) > 64 << 20
    x, w, y = _inputs(T, V, d, dtype, seed=T)
    w[-1] *= 2
    with torch.no_grad():
        out = linear_log_probs(x, w, y, top_k=top)
        _check_forward(out, x, w, y, 1.0, top)
        for a, b in ((8192, T), (8100, 8300)):                            # other rows in the same and in other products
            part = linear_log_probs(x[a:b], w, y[a:b], top_k=top)
            assert torch.equal(part.top_ids, out.top_ids[a:b]) and torch.equal(part.log_probs, out.log_probs[a:b])
    assert _lib.load().swx_device_wait_status() == _lib.SWX_OK
