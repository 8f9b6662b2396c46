"""More language-model operators of this package as measurable passes: log probabilities of given
tokens with the entropy and the top alternatives (from the head's operands, with gradients, and
from logits), and distillation from a teacher's top logits.

``own`` chooses what ``run`` does: False computes each operator in its plain form
(elementary torch operations in fp32, the order of the alternatives' logits in fp64); True calls the
package.  ``exact`` restates each operator in float64 from its definition.
"""
import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # policy-gradient step of the byte-level LM (16 x 512 tokens, d_model 256, 256 bytes): small products, launch-bound
        dict(name="score train bytes", op="score", tokens=8192, vocab=256, dim=256, dtype="bf16", top=0, temp=1.0, train=True, ignored=0.0),
        # the same on a sub-word vocabulary at the decode configuration's width, padding left out
        dict(name="score train large", op="score", tokens=8192, vocab=50001, dim=1024, dtype="bf16", top=0, temp=1.0, train=True, ignored=0.02),
        # fp32, odd sizes, a sampling temperature, the alternatives kept for inspection while training
        dict(name="score train fp32 odd", op="score", tokens=1003, vocab=10007, dim=200, dtype="fp32", top=7, temp=0.7, train=True, ignored=0.1),
        # a teacher scoring a batch: its top alternatives are what a student is trained on
        dict(name="score teacher", op="score", tokens=4096, vocab=50001, dim=1024, dtype="bf16", top=32, temp=1.0, train=False, ignored=0.02),
        # a prompt of bytes scored with alternatives: more than a twentieth of the vocabulary is kept
        dict(name="score bytes", op="score", tokens=512, vocab=256, dim=256, dtype="bf16", top=20, temp=1.0, train=False, ignored=0.0),
        # one token's alternatives from the last hidden state: the weight is the traffic
        dict(name="score single", op="score", tokens=1, vocab=50001, dim=1024, dtype="bf16", top=5, temp=1.0, train=False, ignored=0.0),
        # a student of the byte-level LM on half the vocabulary's mass
        dict(name="distill bytes", op="distill", tokens=8192, vocab=256, dim=256, dtype="bf16", entries=16, temp=1.0, ragged=False),
        # a student on a sub-word vocabulary, softened, some rows padding and some cut short (top-p lists)
        dict(name="distill large", op="distill", tokens=8192, vocab=50001, dim=1024, dtype="bf16", entries=32, temp=2.0, ragged=True),
        # fp32, odd sizes
        dict(name="distill fp32 odd", op="distill", tokens=1003, vocab=10007, dim=200, dtype="fp32", entries=7, temp=1.3, ragged=True),
        # generation: the decode configuration's 256 rows, fp32 logits, what a serving program reports for each token
        dict(name="token batch", op="token", rows=256, vocab=50001, dtype="fp32", top=20, temp=1.0, allowed=1.0),
        # one interactive row of the byte-level LM: latency only
        dict(name="token single", op="token", rows=1, vocab=256, dtype="fp32", top=5, temp=1.0, allowed=1.0),
        # a few rows of bf16 logits (many equal), words forbidden by a grammar, a sampling temperature
        dict(name="token masked odd", op="token", rows=19, vocab=10007, dtype="bf16", top=8, temp=0.7, allowed=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "score", "distill", "token"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    vocab = _log(rng, 65, 50001)
    temp = rng.choice([1.0, 1.0, round(rng.uniform(0.5, 2.0), 2)])
    if op == "token":
        rows = max(1, min(_log(rng, 1, 8192), 256 * 50001 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, top=rng.choice([0, 1, rng.randint(1, 64)]), temp=temp,
                    allowed=rng.choice([1.0, 1.0, 0.999]))
    tokens, dim = _log(rng, 1, 8192), rng.choice([rng.randint(1, 40) * 8, rng.randint(16, 1024), 256, 512, 1024])
    if op == "distill":
        return dict(op=op, tokens=tokens, vocab=vocab, dim=dim, dtype=dtype, entries=_log(rng, 1, 64), temp=temp,
                    ragged=rng.random() < 0.5)
    top = rng.choice([0, rng.randint(1, 64)])
    if top:
        tokens = max(1, min(tokens, 4096 * 50001 // vocab))
    return dict(op=op, tokens=tokens, vocab=vocab, dim=dim, dtype=dtype, top=top, temp=temp, train=rng.random() < 0.5,
                ignored=rng.choice([0.0, 0.05, 0.3]))


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "token":
        r, v, k = case["rows"], case["vocab"], case["top"]
        # the logits, the targets; both values of each row and the alternatives.  A maximum, an exponential and two sums for each logit
        return {"bytes": r * v * es + r * 16 + r * k * 12, "flops": 6.0 * r * v}
    t, v, d = case["tokens"], case["vocab"], case["dim"]
    read = (t * d + v * d) * es
    if case["op"] == "distill":
        # the logits, and each operand's gradient: three products
        return {"bytes": 2 * read + t * case["entries"] * 12 + 4, "flops": 6.0 * t * v * d}
    moved = read + t * 16 + t * case["top"] * 12
    if not case["train"]:
        return {"bytes": moved, "flops": 2.0 * t * v * d}
    return {"bytes": moved + read + t * 8, "flops": 6.0 * t * v * d}


def _rand(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    v = case["vocab"]
    s = dict(case=case)
    if case["op"] == "token":
        r = case["rows"]
        z = _rand(g, (r, v), dt, 2.5)
        y = torch.randint(0, v, (r,), generator=g, device=DEV)
        if case["allowed"] < 1.0:                              # words that a grammar forbids; the token asked for is allowed
            off = torch.rand(r, v, generator=g, device=DEV) >= case["allowed"]
            off.scatter_(1, y[:, None], False)
            off[:, :min(v, case["top"])] = False                # at least as many words as alternatives
            z = z.masked_fill(off, -math.inf)
        return dict(s, z=z, y=y, top=min(case["top"], v))
    t, d = case["tokens"], case["dim"]
    x = _rand(g, (t, d), dt)                                   # the final norm's output
    w = _rand(g, (v, d), dt, 2.5 / math.sqrt(d))
    if case["op"] == "distill":
        k = min(case["entries"], v)
        # k different words a row, the teacher's logits in falling order
        step = torch.randint(1, v // k + 1, (t, 1), generator=g, device=DEV)
        first = torch.randint(0, v, (t, 1), generator=g, device=DEV)
        ids = (first + step * torch.arange(k, device=DEV)) % v
        logits = _rand(g, (t, k), std=2.5).sort(1, descending=True).values
        if case["ragged"]:
            used = torch.randint(1, k + 1, (t, 1), generator=g, device=DEV)
            used = torch.where(torch.rand(t, 1, generator=g, device=DEV) < 0.02, torch.zeros_like(used), used)
            used[0] = k
            ids = torch.where(torch.arange(k, device=DEV) < used, ids, torch.full_like(ids, -1))
        return dict(s, x=x.requires_grad_(), w=w.requires_grad_(), ids=ids, logits=logits)
    y = torch.randint(0, v, (t,), generator=g, device=DEV)
    if case["ignored"] and t > 1:
        drop = torch.rand(t, generator=g, device=DEV) < case["ignored"]
        drop[0] = False
        y = torch.where(drop, torch.full_like(y, -100), y)
    s.update(x=x, w=w, y=y, top=min(case["top"], v))
    if case["train"]:
        x.requires_grad_(), w.requires_grad_()
        # an advantage for each token, and a bonus for the entropy
        s.update(g=_rand(g, (t,), std=1.0 / t), h=_rand(g, (t,), std=0.1 / t))
    return s


def _top(z, k, live=None):
    """The k largest of each row, the lowest index first among equals: (values, indices)."""
    vals, ids = torch.sort(z, dim=1, descending=True, stable=True)
    vals, ids = vals[:, :k].contiguous(), ids[:, :k].contiguous()
    if live is not None:
        vals, ids = torch.where(live[:, None], vals, torch.zeros_like(vals)), torch.where(live[:, None], ids, torch.full_like(ids, -1))
    return vals, ids


def _score_plain(z, y, temp):
    """(log probability of y, entropy) of each row of fp32 logits; zeros where y is -100."""
    z = z / temp
    top = z.detach().amax(1, keepdim=True)
    logp = (z - top) - (z - top).exp().sum(1, keepdim=True).log()
    live = y != -100
    hit = logp.gather(1, torch.where(live, y, torch.zeros_like(y))[:, None])[:, 0]
    terms = logp.exp() * torch.where(logp == -math.inf, torch.zeros_like(logp), logp)
    zero = torch.zeros_like(hit)
    return torch.where(live, hit, zero), torch.where(live, -terms.sum(1), zero), logp


def _distill_plain(x, w, ids, logits, temp):
    z = (x.float() @ w.float().t()) / temp
    top = z.detach().amax(1, keepdim=True)
    lse = (z - top).exp().sum(1, keepdim=True).log() + top
    used = ids >= 0
    t = torch.where(used, logits.float() / temp, torch.full_like(logits, -math.inf, dtype=torch.float32))
    most = t.amax(1, keepdim=True)
    live = most[:, 0] > -math.inf
    e = torch.where(used, (t - torch.where(live[:, None], most, torch.zeros_like(most))).exp(), torch.zeros_like(t))
    q = e / torch.where(live[:, None], e.sum(1, keepdim=True), torch.ones_like(most))
    logq = torch.where(q > 0, q, torch.ones_like(q)).log()
    rows = (q * (logq - (z.gather(1, ids.clamp(min=0)) - lse))).sum(1)
    return (temp * temp) * (torch.where(live, rows, torch.zeros_like(rows)).double().sum() / live.sum()).float()


def _own(s):
    case = s["case"]
    if case["op"] == "token":
        from swiftx_b200.log_probs import token_log_probs
        return token_log_probs(s["z"], s["y"], top_k=s["top"], temperature=case["temp"])
    from swiftx_b200.log_probs import linear_log_probs
    return linear_log_probs(s["x"], s["w"], s["y"], top_k=s["top"], temperature=case["temp"])


def _plain(s):
    case = s["case"]
    top, temp = s["top"], case["temp"]
    if case["op"] == "token":
        lp, ent, logp = _score_plain(s["z"].float(), s["y"], temp)
        ids = _top(s["z"], top)[1] if top else None
        return lp, ent, logp.gather(1, ids) if top else None, ids
    lp, ent, logp = _score_plain(s["x"].float() @ s["w"].float().t(), s["y"], temp)
    if not top:
        return lp, ent, None, None
    live = s["y"] != -100
    # the order of logits that are nearly equal takes 64 bits
    ids = _top(s["x"].detach().double() @ s["w"].detach().double().t(), top, live)[1]
    vals = logp.detach().gather(1, ids.clamp(min=0))
    return lp, ent, torch.where(live[:, None], vals, torch.zeros_like(vals)), ids


def run(state):
    s = state
    case = s["case"]
    if case["op"] == "distill":
        if own:
            from swiftx_b200.loss import linear_distillation
            loss = linear_distillation(s["x"], s["w"], s["ids"], s["logits"], temperature=case["temp"])
        else:
            loss = _distill_plain(s["x"], s["w"], s["ids"], s["logits"], case["temp"])
        dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]))
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    train = case["op"] == "score" and case["train"]
    with torch.set_grad_enabled(train):
        lp, ent, vals, ids = _own(s) if own else _plain(s)
    out = {"log_probs": lp.detach(), "entropy": ent.detach()}
    if s["top"]:
        out.update(top_log_probs=vals, top_ids=ids)
    if train:
        out["dx"], out["dw"] = torch.autograd.grad((lp, ent), (s["x"], s["w"]), (s["g"], s["h"]))
    return out


def _first_largest(z, k):
    """The k largest of each row one after the other, the lowest index of the largest value each time."""
    z, index = z.clone(), torch.arange(z.shape[1], device=z.device)
    left, ids = torch.ones_like(z, dtype=torch.bool), []
    for _ in range(k):
        best = torch.where(left, z, -math.inf).amax(1, keepdim=True)
        at = torch.where(left & (z == best), index, z.shape[1]).amin(1, keepdim=True)
        left.scatter_(1, at, False)
        ids.append(at)
    return torch.cat(ids, 1)


def exact(case, seed):
    s = prepare(case, seed)
    up = lambda t: t.detach().double().requires_grad_(t.requires_grad)  # noqa: E731
    temp = case["temp"]
    if case["op"] == "distill":
        x, w = up(s["x"]), up(s["w"])
        ids, live = s["ids"], (s["ids"] >= 0).any(1)
        t = torch.where(ids >= 0, s["logits"].double() / temp, -math.inf)[live]
        q = torch.softmax(t, 1)
        logp = torch.log_softmax(F.linear(x, w) / temp, 1)[live]
        loss = temp ** 2 * (torch.special.xlogy(q, q) - q * logp.gather(1, ids[live].clamp(min=0))).sum() / live.sum()
        dx, dw = torch.autograd.grad(loss, (x, w))
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    train = case["op"] == "score" and case["train"]
    x, w = (None, None) if case["op"] == "token" else (up(s["x"]), up(s["w"]))
    z = s["z"].double() if x is None else F.linear(x, w)
    y, top = s["y"], s["top"]
    dist = torch.distributions.Categorical(logits=z / temp, validate_args=False)
    live = y != -100
    hit = torch.where(live, dist.logits.gather(1, torch.where(live, y, 0)[:, None])[:, 0], 0.0)
    ent = torch.where(live, torch.special.entr(dist.probs).sum(1), 0.0)
    out = {"log_probs": hit.detach(), "entropy": ent.detach()}
    if top:
        ids = _first_largest(z.detach(), top)
        vals = dist.logits.detach().gather(1, ids)
        out.update(top_log_probs=torch.where(live[:, None], vals, 0.0), top_ids=torch.where(live[:, None], ids, -1))
    if train:
        out["dx"], out["dw"] = torch.autograd.grad((hit, ent), (x, w), (s["g"].double(), s["h"].double()))
    return out
