"""linear_distillation (swx_distill_fwd / _bwd) against float64, and with the scoring that feeds it.

Tolerances.  e_t, E and the dlogit's rounding as for linear_log_probs: a logit is off by e_t = (d / 16 + 8) 2^-23 max_v m_tv
(twice that for fp32 operands), statistics by E = 2^-16 of 1 and the sizes of what is added.  With the temperature tau:
a row's loss is tau^2 sum q (log q - l), off by tau^2 (2 e / tau + E (1 + sum q (|log q| + |l|) + H)).
dz = tau c (p - Q), Q the teacher's share of a word: p is off by 2 e / tau + E of itself, Q by 2^-18 of
itself; then one rounding to bf16 (2^-8; 2^-22 for fp32 operands) and the products as for the loss.
"""
import math

import pytest
import torch

from swiftx_b200 import _lib
from swiftx_b200.log_probs import linear_log_probs, token_log_probs
from swiftx_b200.loss import linear_cross_entropy, linear_distillation
from swiftx_b200.sift import SiftConfig, SiftLM

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32
E = 2.0 ** -16


def _inputs(T, V, d, K, dtype, seed=0, t_dtype=FP):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, d, generator=g, device=DEV).to(dtype)
    w = (torch.randn(V, d, generator=g, device=DEV) * 2 / d ** 0.5).to(dtype)
    ids = torch.rand(T, V, generator=g, device=DEV).topk(K, 1).indices
    logits = (torch.randn(T, K, generator=g, device=DEV) * 2).to(t_dtype)
    return x, w, ids, logits


def _exact(x, w, ids, logits, temp):
    """(row losses, p, Q as a (T, V) matrix, live, q, l at the entries) in float64."""
    z = x.double() @ w.double().t()
    l = torch.log_softmax(z / temp, 1)
    used = (ids >= 0) & (logits > -math.inf)
    live = used.any(1)
    q = torch.softmax(torch.where(used, logits.double() / temp, -math.inf).masked_fill(~live[:, None], 0.0), 1)
    q = torch.where(used, q, 0.0)
    at = l.gather(1, ids.clamp(min=0))
    rows = temp ** 2 * torch.where(used, torch.special.xlogy(q, q) - q * at, 0.0).sum(1)
    Q = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), q)
    return rows, l, Q, live, q, at


def _run(x, w, ids, logits, temp=1.0, reduction="mean", dloss=None):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_distillation(x, w, ids, logits, temperature=temp, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss) if dloss is None else dloss)
    assert _lib.load().swx_device_wait_status() == _lib.SWX_OK
    return loss.detach(), dx, dw


def _check(x, w, ids, logits, temp, reduction, loss, dx, dw, dloss=None):
    T, d = x.shape
    bf = x.dtype == BF
    xd, wd = x.double(), w.double()
    e = (d / 16 + 8) * 2.0 ** -23 * (xd.abs() @ wd.abs().t()).amax(1) * (1 if bf else 2) / temp
    rows, l, Q, live, q, at = _exact(x, w, ids, logits, temp)
    p = l.exp()
    H = -(p * l).sum(1)
    size = 1 + H + (q * at.abs() - torch.special.xlogy(q, q)).sum(1)
    row_bound = torch.where(live, temp ** 2 * (2 * e + E * size), 0.0)
    c = (torch.ones(T, device=DEV) if dloss is None else dloss).double().expand(T)
    if reduction == "none":
        want, bound = rows, row_bound
    else:
        n = live.sum() if reduction == "mean" else 1
        want, bound = rows.sum() / n, row_bound.sum() / n + 2.0 ** -23 * (rows.sum() / n).abs()
        c = c / n
    assert bool(((loss.double() - want).abs() <= bound).all()), float(((loss.double() - want).abs() / bound).max())
    c = torch.where(live, c, 0.0) * temp
    dz = c[:, None] * (p - Q)
    off = c.abs()[:, None] * ((2 * e + E)[:, None] * p + 2.0 ** -18 * Q)
    r = 2.0 ** -8 if bf else 2.0 ** -22
    for got, a, o, other, n in ((dx, dz, off, wd, w.shape[0]), (dw, dz.t(), off.t(), xd, T)):
        want = a @ other
        bound = 1.02 * (((r + (n / 16 + 16) * 2.0 ** -23) * a.abs() + 1.02 * o) @ other.abs())
        if got.dtype == BF:
            bound = bound + 2.0 ** -8 * want.abs()
        err = (got.double() - want).abs()
        assert bool((err <= bound + 1e-38).all()), f"largest error over bound {float((err / (bound + 1e-38)).max()):.3g}"


@pytest.mark.parametrize("T,V,d,K,dtype,temp,reduction", [
    (1, 1, 1, 1, BF, 1.0, "mean"), (1, 65, 17, 65, BF, 2.0, "sum"), (5, 300, 8, 3, FP, 1.0, "none"), (256, 256, 64, 16, BF, 1.0, "mean"),
    (257, 257, 65, 33, BF, 0.5, "none"), (300, 513, 200, 7, FP, 3.0, "mean"), (1000, 1003, 256, 128, BF, 1.0, "sum"),
    (33, 5001, 40, 100, FP, 1.5, "sum"), (130, 3001, 1030, 32, BF, 1.0, "mean"), (600, 2000, 100, 5, FP, 2.0, "none"), (40, 700, 1030, 20, FP, 1.0, "mean"),
])
def test_loss_and_gradients(T, V, d, K, dtype, temp, reduction):
    x, w, ids, logits = _inputs(T, V, d, K, dtype, seed=T + V)
    dloss = torch.randn(T, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) if reduction == "none" else None
    _check(x, w, ids, logits, temp, reduction, *_run(x, w, ids, logits, temp, reduction, dloss), dloss)


def test_several_pieces_of_the_vocabulary():
    for T, V, d, dtype in ((12288, 20000, 72, BF), (9000, 9001, 40, FP)):
        x, w, ids, logits = _inputs(T, V, d, 9, dtype, seed=3)
        _check(x, w, ids, logits, 1.0, "mean", *_run(x, w, ids, logits))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_unused_entries_and_empty_rows(dtype):
    x, w, ids, logits = _inputs(90, 400, 40, 12, dtype, seed=5)
    ids[::3, 5:] = -1                                                     # cut short
    logits[1::3, ::2] = -math.inf                                         # dropped by their logits
    logits[0, 5:] = math.nan                                              # whatever stands in an unused entry
    ids[7] = -100
    logits[8] = -math.inf
    for red in ("mean", "sum", "none"):
        got = _run(x, w, ids, logits.nan_to_num(0.0, neginf=-math.inf) if red == "sum" else logits, 1.3, red)
        clean = torch.where(ids < 0, 0.0, logits)
        _check(x, w, ids, clean, 1.3, red, *got)
        assert not got[1][7].any() and not got[1][8].any()
        if red == "none":
            assert float(got[0][7]) == float(got[0][8]) == 0.0
    empty = torch.full_like(ids, -1)
    loss, dx, dw = _run(x, w, empty, logits)
    assert torch.isnan(loss) and not dx.any() and not dw.any()
    loss, dx, dw = _run(x, w, empty, logits, reduction="sum")
    assert float(loss) == 0.0 and not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_the_same_word_in_several_entries(dtype):
    x, w, ids, logits = _inputs(70, 300, 24, 40, dtype, seed=6)
    ids[:, 35] = ids[:, 2]
    ids[:, 36] = ids[:, 2]
    ids[5] = 17
    ids[6, 1::2] = -1
    _check(x, w, ids, logits, 1.0, "mean", *_run(x, w, ids, logits))


def test_one_sure_word_is_the_cross_entropy():
    """A teacher with a single word gives the loss of that target; gradients by the same kernels but for the word's own logit."""
    x, w, _, _ = _inputs(120, 777, 64, 1, FP, seed=7)
    y = torch.randint(0, 777, (120,), device=DEV)
    y[::5] = -100
    a = _run(x, w, y[:, None], torch.zeros(120, 1, device=DEV))
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(xr, wr, y)
    b = (loss, *torch.autograd.grad(loss, (xr, wr)))
    tol = 2.0 ** -14                                                     # E on either side, a few times
    for p, q in zip(a, b):
        assert float((p - q).norm()) <= tol * float(q.norm())


def test_bad_entries_are_loud():
    x, w, ids, logits = _inputs(80, 300, 32, 6, FP, seed=8)
    base = _run(x, w, ids, logits, reduction="none")
    for change in (lambda i, t: i[4].__setitem__(2, 300), lambda i, t: i[4].__setitem__(2, 1 << 40), lambda i, t: t[4].__setitem__(1, math.nan),
                   lambda i, t: t[4].__setitem__(1, math.inf)):
        i, t = ids.clone(), logits.clone()
        change(i, t)
        loss, dx, dw = _run(x, w, i, t, reduction="none")
        assert torch.isnan(loss[4]) and torch.isnan(dx[4]).all()
        assert torch.equal(loss[5:], base[0][5:]) and torch.equal(dx[5:], base[1][5:])
        assert torch.isnan(_run(x, w, i, t)[0])


def test_against_differences():
    """A central difference of the operator is off by its values' errors over the step, and from the derivative by what
    float64 says the step makes."""
    T, V, d, K, temp = 40, 200, 24, 9, 1.5
    x, w, ids, logits = _inputs(T, V, d, K, FP, seed=9)
    u, v = torch.randn_like(x) / 8, torch.randn_like(w) / 8
    _, dx, dw = _run(x, w, ids, logits, temp, "sum")
    got = float((dx.double() * u).sum() + (dw.double() * v).sum())
    step = 2.0 ** -4
    f64 = lambda t: float(_exact(x + t * u, w + t * v, ids, logits, temp)[0].sum())  # noqa: E731
    f = lambda t: float(linear_distillation(x + t * u, w + t * v, ids, logits, temperature=temp, reduction="sum"))  # noqa: E731
    diff, diff64 = (f(step) - f(-step)) / (2 * step), (f64(step) - f64(-step)) / (2 * step)
    rows, l, Q, live, q, at = _exact(x, w, ids, logits, temp)
    dz = temp * (l.exp() - Q)
    exact = float(((dz @ w.double()) * u).sum() + ((dz.t() @ x.double()) * v).sum())
    e = 1.5 * 2 * (d / 16 + 8) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()).amax(1) / temp
    noise = float((temp ** 2 * (2 * e + 2 * E * (8 + q.mul(at.abs()).sum(1)))).sum())
    assert abs(diff - diff64) <= noise / step
    assert abs(got - diff) <= abs(exact - diff64) + noise / step + 2.0 ** -12 * float(((dz @ w.double()) * u).abs().sum() + ((dz.t() @ x.double()) * v).abs().sum())


def test_layouts_types_and_partial_gradients():
    T, V, d, K = 160, 700, 64, 10
    x, w, ids, logits = _inputs(T, V, d, K, BF, seed=10, t_dtype=BF)
    base = _run(x, w, ids, logits)
    _check(x, w, ids, logits, 1.0, "mean", *base)
    wide = torch.zeros(T, 2 * d, device=DEV, dtype=BF)
    wide[:, d:] = x
    odd_w = torch.zeros(V, d + 1, device=DEV, dtype=BF)
    odd_w[:, 1:] = w
    ids2, logits2 = torch.full((T, 2 * K + 1), -7, device=DEV), torch.zeros(T, 2 * K + 1, device=DEV, dtype=BF)
    ids2[:, 1:K + 1], logits2[:, K + 1:] = ids, logits
    for args in ((wide[:, d:], w, ids, logits), (x, odd_w[:, 1:], ids, logits), (x, w, ids2[:, 1:K + 1], logits2[:, K + 1:]),
                 (x.t().contiguous().t(), w.t().contiguous().t(), ids.t().contiguous().t(), logits.float())):
        for a, b in zip(base, _run(*args)):
            assert torch.equal(a, b)
    same = torch.randint(0, V, (1, K), device=DEV).expand(T, K)           # one list for every row
    for a, b in zip(_run(x, w, same, logits[:1].expand(T, K)), _run(x, w, same.contiguous(), logits[:1].repeat(T, 1))):
        assert torch.equal(a, b)
    shaped = linear_distillation(x.view(4, 40, d), w, ids.view(4, 40, K), logits.view(4, 40, K), reduction="none")
    assert shaped.shape == (4, 40) and torch.equal(shaped.view(-1), linear_distillation(x, w, ids, logits, reduction="none"))
    for on in ((True, False), (False, True)):
        xr, wr = x.detach().requires_grad_(on[0]), w.detach().requires_grad_(on[1])
        linear_distillation(xr, wr, ids, logits).backward()
        for g, b, want in zip((xr.grad, wr.grad), base[1:], on):
            assert (g is None) == (not want) and (g is None or torch.equal(g, b))
    with torch.no_grad():
        assert torch.equal(linear_distillation(x, w, ids, logits), base[0])


def test_fp32_weight_with_bf16_input_and_autocast():
    x, w, ids, logits = _inputs(260, 900, 80, 6, FP, seed=4)
    x16 = x.to(BF)
    loss, dx, dw = _run(x16, w, ids, logits)
    assert dw.dtype == FP and dx.dtype == BF
    _check(x16, w.to(BF), ids, logits, 1.0, "mean", loss, dx, dw)
    with torch.autocast("cuda", dtype=BF):
        a = _run(x, w, ids, logits)
    assert torch.equal(a[0], loss) and torch.equal(a[2], dw) and a[1].dtype == FP


def test_no_tokens():
    w = torch.randn(50, 16, device=DEV, requires_grad=True)
    x = torch.zeros(0, 16, device=DEV, requires_grad=True)
    ids, logits = torch.zeros(0, 3, device=DEV, dtype=torch.int64), torch.zeros(0, 3, device=DEV)
    assert torch.isnan(linear_distillation(x, w, ids, logits))
    linear_distillation(x, w, ids, logits, reduction="sum").backward()
    assert not w.grad.any() and x.grad.shape == (0, 16)
    assert linear_distillation(x, w, ids, logits, reduction="none").shape == (0,)


def test_deterministic_streams_and_graphs():
    x, w, ids, logits = _inputs(1003, 3001, 72, 20, BF, seed=6)
    a = _run(x, w, ids, logits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _run(x, w, ids, logits)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    graphs = []
    for s in (6, 7):
        xs, ws, i, t = _inputs(300, 2001, 72, 9, BF, seed=s)
        xs.requires_grad_(), ws.requires_grad_()

        def f(xs=xs, ws=ws, i=i, t=t):
            loss = linear_distillation(xs, ws, i, t)
            return [loss.detach(), *torch.autograd.grad(loss, (xs, ws))]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = f()
        graphs.append((xs, t, f, graph, r))
    for xs, t, *_ in graphs:
        with torch.no_grad():
            xs.mul_(0.5), t.mul_(2)
    for *_, graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, _, f, _, r in graphs:
        for p, q in zip([t.clone() for t in r], f()):
            assert torch.equal(p, q)


def test_refusals():
    x, w, ids, logits = _inputs(10, 20, 16, 4, BF)
    for args in ((x, w[:, :8], ids, logits), (x, w, ids[:5], logits), (x, w, ids, logits[:, :3]), (x, w, ids.int(), logits), (x, w, ids, logits.double()),
                 (x, w, ids[:, 0], logits[:, 0]), (x, w, ids[:, :0], logits[:, :0]), (x, w, ids.repeat(1, 33), logits.repeat(1, 33)),
                 (x.float(), w, ids, logits), (x.double(), w.double(), ids, logits), (x, w, ids[None], logits[None])):
        with pytest.raises(ValueError):
            linear_distillation(*args)
    for kw in (dict(reduction="max"), dict(temperature=0.0), dict(temperature=-2.0), dict(temperature=math.nan)):
        with pytest.raises(ValueError):
            linear_distillation(x, w, ids, logits, **kw)
    with pytest.raises(RuntimeError, match="not differentiable"):
        linear_distillation(x, w, ids, logits.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        linear_distillation(x.cpu(), w.cpu(), ids.cpu(), logits.cpu())


def test_transforms():
    from torch.autograd import forward_ad
    x, w, ids, logits = _inputs(50, 90, 24, 4, FP)
    with forward_ad.dual_level():
        for which in (0, 1):
            pair = [x, w]
            pair[which] = forward_ad.make_dual(pair[which], torch.ones_like(pair[which]))
            with pytest.raises(NotImplementedError):
                linear_distillation(*pair, ids, logits)
        with pytest.raises(RuntimeError, match="not differentiable"):
            linear_distillation(x, w, ids, forward_ad.make_dual(logits, torch.ones_like(logits)))
    f = torch.jit.trace(lambda x, w: linear_distillation(x, w, ids, logits, reduction="none"), (x, w))
    x2, w2, _, _ = _inputs(50, 90, 24, 4, FP, seed=1)
    assert torch.equal(f(x2, w2), linear_distillation(x2, w2, ids, logits, reduction="none"))


# ------------------------------------------------------------------ together, as a program uses them
@pytest.mark.parametrize("autocast", [False, True])
def test_teacher_to_student(autocast):
    """A teacher scores a padded batch, its alternatives go to the student's loss as they are (ids of -1 where the targets were
    ignored); the student's gradients are those of the loss through its logits.  Tolerances as for SiftLM.loss against forward's:
    2^-12 of each norm in fp32, 4 * 2^-8 under autocast, where forward rounds the logits to bf16."""
    torch.manual_seed(0)
    teacher = SiftLM(SiftConfig(vocab_size=300, d_model=96, n_layers=2)).to(DEV)
    student = SiftLM(SiftConfig(vocab_size=300, d_model=64, n_layers=2)).to(DEV)
    with torch.no_grad():
        for m in (teacher, student):
            m.embedding.weight.mul_(10)
    idx, tgt = torch.randint(0, 300, (3, 50), device=DEV), torch.randint(0, 300, (3, 50), device=DEV)
    tgt[1, 40:] = -100
    tol = 4 * 2.0 ** -8 if autocast else 2.0 ** -12
    with torch.no_grad(), torch.autocast("cuda", dtype=BF, enabled=autocast):
        scored = teacher.log_probs(idx, tgt, top_k=8)
        logits = teacher(idx)[0].double()
    l = torch.log_softmax(logits, -1)
    live = tgt != -100
    want = torch.where(live, l.gather(2, tgt.clamp(min=0)[..., None])[..., 0], 0.0)
    assert float((scored.log_probs.double() - want).norm()) <= tol * float(want.norm())
    assert bool((scored.top_ids[~live] == -1).all()) and bool((scored.top_ids[live] >= 0).all())
    got = []
    temp = 2.0
    for plain in (True, False):
        student.zero_grad()
        with torch.autocast("cuda", dtype=BF, enabled=autocast):
            if plain:
                ls = torch.log_softmax(student(idx)[0].float() / temp, -1)[live]
                q = torch.softmax(scored.top_log_probs[live] / temp, -1)
                loss = temp ** 2 * (q * (q.log() - ls.gather(1, scored.top_ids[live]))).sum() / live.sum()
            else:
                loss = student.distillation_loss(idx, scored.top_ids, scored.top_log_probs, temperature=temp)
        loss.backward()
        got.append((float(loss.detach()), {n: p.grad.clone() for n, p in student.named_parameters()}))
    assert abs(got[0][0] - got[1][0]) <= tol * abs(got[0][0])
    for n, g in got[0][1].items():
        assert float((g - got[1][1][n]).norm()) <= 2 * tol * float(g.norm()) + 1e-7, n


def test_policy_gradient_of_the_model():
    """log_probs' gradient through the whole model against the one through forward's logits (fp32: 2^-12 of each norm)."""
    torch.manual_seed(1)
    model = SiftLM(SiftConfig(vocab_size=200, d_model=64, n_layers=2)).to(DEV)
    with torch.no_grad():
        model.embedding.weight.mul_(10)
    idx, tgt = torch.randint(0, 200, (2, 40), device=DEV), torch.randint(0, 200, (2, 40), device=DEV)
    adv = torch.randn(2, 40, device=DEV)
    got = []
    for plain in (True, False):
        model.zero_grad()
        if plain:
            l = torch.log_softmax(model(idx)[0], -1)
            lp, ent = l.gather(2, tgt[..., None])[..., 0], -(l.exp() * l).sum(-1)
        else:
            lp, ent, _, _ = model.log_probs(idx, tgt)
        (-(adv * lp).mean() - 0.1 * ent.mean()).backward()
        got.append({n: p.grad.clone() for n, p in model.named_parameters()})
    for n, g in got[0].items():
        assert float((g - got[1][n]).norm()) <= 2.0 ** -12 * float(g.norm()) + 1e-7, n


@pytest.mark.parametrize("graphed", [False, True])
def test_generation_reports_what_scoring_finds(graphed):
    """generate's log probabilities of its tokens are those of scoring the text that it wrote (the recurrent and the
    sequence forms of the model, fp32: 2^-10 of logits of some units)."""
    torch.manual_seed(2)
    model = SiftLM(SiftConfig(vocab_size=120, d_model=64, n_layers=2)).to(DEV)
    with torch.no_grad():
        model.embedding.weight.mul_(10)
    prompt = torch.randint(0, 120, (3, 7), device=DEV)
    text, scores = model.generate(prompt, 9, temperature=0.8, top_k=30, graphed=graphed, log_probs=4)
    assert text.shape == (3, 16) and scores.log_probs.shape == scores.entropy.shape == (3, 9) and scores.top_ids.shape == (3, 9, 4)
    with torch.no_grad():
        again = model.log_probs(text[:, :-1], text[:, 1:], top_k=4)
        direct = token_log_probs(model(text[:, :-1])[0], text[:, 1:], top_k=4)
    for a, b, c in zip(scores[:3], again[:3], direct[:3]):
        assert float((a - b[:, 6:]).abs().max()) <= 2.0 ** -10 * (1 + float(b.abs().max()))
        assert float((c - b).abs().max()) <= 2.0 ** -10 * (1 + float(b.abs().max()))
    text, scores = model.generate(prompt, 2, temperature=0, log_probs=0)
    assert scores.top_ids is None and bool((scores.log_probs <= 0).all())
    assert torch.equal(model.generate(prompt, 2, temperature=0), text)
    text, scores = model.generate(prompt, 0, log_probs=2)
    assert torch.equal(text, prompt) and scores.log_probs.shape == (3, 0) and scores.top_ids.shape == (3, 0, 2)


def test_two_scorings_at_once_on_two_streams():
    x, w, ids, logits = _inputs(500, 4001, 64, 8, BF, seed=12)
    y = ids[:, 0].contiguous()
    want = [*linear_log_probs(x, w, y, top_k=6), linear_distillation(x, w, ids, logits)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([*linear_log_probs(x, w, y, top_k=6), linear_distillation(x, w, ids, logits)])
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T,V,d,K,dtype", [(8193, 300, 24, 3, BF), (17000, 260, 32, 20, BF), (16391, 700, 40, 40, FP)])
def test_more_rows_than_one_product_takes(T, V, d, K, dtype):
    x, w, ids, logits = _inputs(T, V, d, K, dtype, seed=12)
    ids[::5, 1:] = -1
    ids[8190:8195] = -1
    for red in ("mean", "sum", "none"):
        got = _run(x, w, ids, logits, 1.5, red)
        _check(x, w, ids, logits, 1.5, red, *got)
    # rows do not see each other
    for a, b in ((0, 100), (8100, 8300), (T - 50, T)):
        part = _run(x[a:b], w, ids[a:b], logits[a:b], 1.5, "none")
        assert torch.equal(part[0], got[0][a:b])
    xo = torch.zeros(T, d + 3, device=DEV, dtype=dtype)[:, 3:]            # rows off 16 bytes
    xo.copy_(x)
    assert torch.equal(_run(xo, w, ids, logits, 1.5, "none")[0], got[0])


def test_a_width_that_is_not_supported_is_named():
    x, w = torch.zeros(2, 65544, device=DEV, dtype=BF), torch.zeros(3, 65544, device=DEV, dtype=BF)
    ids, logits = torch.zeros(2, 1, device=DEV, dtype=torch.int64), torch.zeros(2, 1, device=DEV)
    with pytest.raises(ValueError, match="swx_distill"):
        linear_distillation(x, w, ids, logits)
    with pytest.raises(ValueError, match="swx_logprob"):
        linear_log_probs(x, w, ids[:, 0])
