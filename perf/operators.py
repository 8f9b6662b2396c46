"""The language-model operators of this package as measurable passes: linear attention with
a decay for each head (over a sequence, with its gradient, and for single tokens) and the
head's softmax cross entropy over a large vocabulary with its gradient.

``own`` chooses what ``run`` does: False computes each operator in its plain form
(elementary torch operations in fp32, rounded once to the output's type); True calls the
package.  ``exact`` restates each operator in float64 from its definition.
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the byte-level LM's own training step (16 x 512 tokens, d_model 256, 256 bytes): small products, launch-bound
        dict(name="loss train bytes", op="loss", tokens=8192, vocab=256, dim=256, dtype="bf16", train=True, ignored=0.0),
        # the same head on a sub-word vocabulary at the decode configuration's width: the step's largest product
        dict(name="loss train large", op="loss", tokens=8192, vocab=50001, dim=1024, dtype="bf16", train=True, ignored=0.02),
        # fp32 training at odd sizes, a tenth of the batch padding
        dict(name="loss train fp32 odd", op="loss", tokens=1003, vocab=10007, dim=200, dtype="fp32", train=True, ignored=0.1),
        # one prompt scored token by token (perplexity of a 512-token row): no gradient, the weight is most of the traffic
        dict(name="loss score", op="loss", tokens=512, vocab=50001, dim=1024, dtype="bf16", train=False, ignored=0.0),
        # one block's training pass at the scan's benchmark shape (8 x 2048, 512 channels as 8 heads of 64)
        dict(name="attention train", op="attention", batch=8, length=2048, heads=8, qk_heads=8, dk=64, dv=64,
             dtype="bf16", decay="token", train=True, state=False, ragged=False),
        # fp32 training, shared query / key heads, odd head sizes and length, a state carried in and out (a long text in pieces)
        dict(name="attention train fp32 odd", op="attention", batch=2, length=777, heads=6, qk_heads=2, dk=40, dv=56,
             dtype="fp32", decay="token", train=True, state=True, ragged=False),
        # a wide state with one shared query / key head and a fixed decay for each head, the LM's batch
        dict(name="attention train shared", op="attention", batch=16, length=512, heads=16, qk_heads=1, dk=128, dv=64,
             dtype="bf16", decay="head", train=True, state=False, ragged=False),
        # a padded batch of prompts of different lengths before generation
        dict(name="attention prompts", op="attention", batch=8, length=1000, heads=16, qk_heads=16, dk=64, dv=128,
             dtype="bf16", decay="token", train=False, state=True, ragged=True),
        # the long-sequence configuration (4 x 65536, 2048 channels as 32 heads of 64)
        dict(name="attention long", op="attention", batch=4, length=65536, heads=32, qk_heads=32, dk=64, dv=64,
             dtype="bf16", decay="token", train=False, state=True, ragged=False),
        # generation, one token a row: the decode configuration (256 rows, 2048 channels)
        dict(name="step batch", op="step", batch=256, heads=32, qk_heads=32, dk=64, dv=64, dtype="bf16", decay="token"),
        # one interactive row: latency only
        dict(name="step single", op="step", batch=1, heads=8, qk_heads=8, dk=64, dv=64, dtype="fp32", decay="token"),
        # a few rows, odd sizes, shared query / key heads and a wide state
        dict(name="step odd", op="step", batch=19, heads=10, qk_heads=5, dk=128, dv=72, dtype="bf16", decay="head"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "attention", "attention", "step"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "loss":
        tokens, dim = _log(rng, 1, 8192), rng.choice([rng.randint(1, 40) * 8, rng.randint(16, 1024), 256, 512, 1024])
        return dict(op=op, tokens=tokens, vocab=_log(rng, 65, 50001), dim=dim, dtype=dtype,
                    train=rng.random() < 0.7, ignored=rng.choice([0.0, 0.05, 0.3]))
    qk_heads = rng.randint(1, 8)
    heads = qk_heads * rng.choice([1, 1, 2, 3])
    dk, dv = (rng.choice([16, 32, 64, 128, rng.randint(1, 128)]) for _ in range(2))
    decay = rng.choice(["token", "token", "head"])
    if op == "step":
        return dict(op=op, batch=_log(rng, 1, 256), heads=heads, qk_heads=qk_heads, dk=dk, dv=dv, dtype=dtype, decay=decay)
    length = _log(rng, 1, 4096)
    return dict(op=op, batch=max(1, min(16, 16384 // length, _log(rng, 1, 16))), length=length, heads=heads, qk_heads=qk_heads,
                dk=dk, dv=dv, dtype=dtype, decay=decay, train=rng.random() < 0.6, state=rng.random() < 0.5,
                ragged=rng.random() < 0.3)


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "loss":
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        read = (t * d + v * d) * es + t * 8
        if not case["train"]:
            return {"bytes": read + t * 4, "flops": 2.0 * t * v * d}
        # the logits, and each operand's gradient: three products
        return {"bytes": read + (t * d + v * d) * es + 4, "flops": 6.0 * t * v * d}
    h, hk, dk, dv = case["heads"], case["qk_heads"], case["dk"], case["dv"]
    if case["op"] == "step":
        rows = case["batch"]
        decay = rows * h * 4 if case["decay"] == "token" else h * 4
        # the state is read and written; update (decay, product, sum) and readout, a multiply and an add each
        return {"bytes": rows * (8.0 * h * dk * dv + es * (2 * hk * dk + 2 * h * dv)) + decay, "flops": 5.0 * rows * h * dk * dv}
    b, n = case["batch"], case["length"]
    rows = b * n
    decay = rows * h * 4 if case["decay"] == "token" else h * 4
    state = b * h * dk * dv * 4
    tensors = rows * (2 * hk * dk + h * dv) * es          # q, k, v
    # the recurrence itself: the state's update and its readout, a multiply and an add for each of its values
    fwd = 4.0 * rows * h * dk * dv
    moved = tensors + rows * h * dv * es + decay + (2 if case["state"] else 0) * state
    if not case["train"]:
        return {"bytes": moved, "flops": fwd}
    moved += tensors + decay + rows * h * dv * es + (2 if case["state"] else 0) * state   # gradients, and the output's
    return {"bytes": moved, "flops": 3 * fwd}


def _rand(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _decay(case, g, shape):
    """-A dt with A in [1, 16] for each head and dt log-uniform in [1e-3, 0.1], as the selective scan's decays."""
    h = case["heads"]
    a = 1 + 15 * torch.rand(h, generator=g, device=DEV)
    if case["decay"] == "head":
        shape = (h,)
    dt = torch.exp(torch.rand(shape, generator=g, device=DEV) * math.log(100.0) + math.log(1e-3))
    return -a * dt


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    if case["op"] == "loss":
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        x = _rand(g, (t, d), dt)                                   # the final norm's output
        w = _rand(g, (v, d), dt, 1.5 / math.sqrt(d))
        y = torch.randint(0, v, (t,), generator=g, device=DEV)
        if case["ignored"] and t > 1:
            drop = torch.rand(t, generator=g, device=DEV) < case["ignored"]
            drop[0] = False
            y = torch.where(drop, torch.full_like(y, -100), y)
        return dict(case=case, x=x.requires_grad_(case["train"]), w=w.requires_grad_(case["train"]), y=y)
    b, h, hk, dk, dv = case["batch"], case["heads"], case["qk_heads"], case["dk"], case["dv"]
    s = dict(case=case, scale=dk ** -0.5)
    if case["op"] == "step":
        s.update(q=_rand(g, (b, hk, dk), dt), k=_rand(g, (b, hk, dk), dt), v=_rand(g, (b, h, dv), dt),
                 g=_decay(case, g, (b, h)), s0=_rand(g, (b, h, dk, dv)))
        return s
    n = case["length"]
    s.update(q=_rand(g, (b, n, hk, dk), dt), k=_rand(g, (b, n, hk, dk), dt), v=_rand(g, (b, n, h, dv), dt),
             g=_decay(case, g, (b, n, h)), s0=_rand(g, (b, h, dk, dv)) if case["state"] else None, lengths=None)
    if case["ragged"]:
        s["lengths"] = torch.randint(0, n + 1, (b,), generator=g, device=DEV)
    if case["train"]:
        for k in ("q", "k", "v", "g", "s0"):
            if s[k] is not None:
                s[k].requires_grad_()
        s["do"] = _rand(g, (b, n, h, dv), dt)
        s["ds"] = _rand(g, (b, h, dk, dv)) if case["state"] else None
    return s


def _attention_plain(q, k, v, g, s0, scale, lengths, chunk=64):
    """The chunked form: decayed scores inside a chunk, and the states at the chunks' starts by
    one product with the chunks' decays.  The decays' sums are in 64 bits (far positions)."""
    b, n, h, dv = v.shape
    hk, dk = q.shape[2], q.shape[3]
    out_dtype = v.dtype
    q, k, v = q.float(), k.float(), v.float()
    g = g.double().expand(b, n, h)
    if lengths is not None:
        live = torch.arange(n, device=v.device)[None, :, None] < lengths[:, None, None]
        q, k, v = (torch.where(live[..., None], t, torch.zeros((), device=v.device)) for t in (q, k, v))
        g = torch.where(live, g, torch.zeros((), device=v.device, dtype=g.dtype))
    c = min(chunk, n)
    nc = -(-n // c)
    fit = lambda t: torch.cat([t, t.new_zeros((b, nc * c - n) + t.shape[2:])], 1).reshape((b, nc, c) + t.shape[2:])  # noqa: E731
    q, k, v = (fit(t).permute(0, 3, 1, 2, 4) for t in (q, k, v))                    # (b, heads, nc, c, d)
    q, k = (t.repeat_interleave(h // hk, 1) for t in (q, k))
    run = fit(g).permute(0, 3, 1, 2).cumsum(-1)                                     # (b, h, nc, c)
    gap = run[..., :, None] - run[..., None, :]
    keep = torch.ones(c, c, device=v.device, dtype=torch.bool).tril()
    inside = torch.where(keep, gap, gap.new_full((), -math.inf)).exp().float()
    out = ((q @ k.transpose(-1, -2)) * inside) @ v
    last = run[..., -1:]
    part = (k * (last - run).exp().float()[..., None]).transpose(-1, -2) @ v        # (b, h, nc, dk, dv)
    total = torch.cat([torch.zeros_like(last[..., :1, 0]), last[..., 0].cumsum(-1)], -1)   # (b, h, nc + 1)
    far = total[..., :, None] - total[..., None, 1:]
    keep = torch.ones(nc + 1, nc, device=v.device, dtype=torch.bool).tril(-1)
    far = torch.where(keep, far, far.new_full((), -math.inf)).exp().float()
    states = (far @ part.flatten(-2)).unflatten(-1, (dk, dv))                       # at each chunk's start, and the end
    if s0 is not None:
        states = states + total.exp().float()[..., None, None] * s0[:, :, None]
    out = out + (q * run.exp().float()[..., None]) @ states[:, :, :-1]
    out = (scale * out).permute(0, 2, 3, 1, 4).reshape(b, nc * c, h, dv)[:, :n]
    return out.to(out_dtype), states[:, :, -1]


def _loss_plain(x, w, y, mean):
    logits = x.float() @ w.float().t()
    top = logits.detach().amax(-1, keepdim=True)
    lse = (logits - top).exp().sum(-1).log() + top[:, 0]
    live = y != -100
    hit = logits.gather(1, torch.where(live, y, torch.zeros_like(y))[:, None])[:, 0]
    rows = torch.where(live, lse - hit, torch.zeros_like(lse))
    return rows.double().sum().div(live.sum()).float() if mean else rows


def _step_plain(q, k, v, g, state, scale):
    h = v.shape[1]
    q, k = (t.float().repeat_interleave(h // t.shape[1], 1) for t in (q, k))
    new = state * g.float().exp().expand(v.shape[0], h)[..., None, None] + k[..., None] * v.float()[:, :, None]
    out = (q[:, :, None] @ new)[:, :, 0] * scale
    state.copy_(new)
    return out.to(v.dtype)


def _grads(s, out, state):
    names = [n for n in ("q", "k", "v", "g", "s0") if s[n] is not None]
    outs, douts = ([out, state], [s["do"], s["ds"]]) if s["ds"] is not None else ([out], [s["do"]])
    return {"d" + n: t for n, t in zip(names, torch.autograd.grad(outs, [s[n] for n in names], douts))}


def run(state):
    s = state
    case = s["case"]
    if case["op"] == "loss":
        if own:
            from swiftx_b200.loss import linear_cross_entropy
            f = lambda: linear_cross_entropy(s["x"], s["w"], s["y"], reduction="mean" if case["train"] else "none")  # noqa: E731
        else:
            f = lambda: _loss_plain(s["x"], s["w"], s["y"], case["train"])  # noqa: E731
        if not case["train"]:
            with torch.no_grad():
                return {"loss": f()}
        loss = f()
        dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]))
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    if case["op"] == "step":
        if own:
            from swiftx_b200.linear_attention import linear_attention_step
            out = linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["s0"], scale=s["scale"])
        else:
            out = _step_plain(s["q"], s["k"], s["v"], s["g"], s["s0"], s["scale"])
        return {"out": out, "state": s["s0"]}
    with torch.set_grad_enabled(case["train"]):
        if own:
            from swiftx_b200.linear_attention import linear_attention
            out = linear_attention(s["q"], s["k"], s["v"], s["g"], initial_state=s["s0"], scale=s["scale"],
                                   lengths=s["lengths"], return_state=case["state"])
            out, last = out if case["state"] else (out, None)
        else:
            out, last = _attention_plain(s["q"], s["k"], s["v"], s["g"], s["s0"], s["scale"], s["lengths"])
            last = last if case["state"] else None
    got = {"out": out.detach(), "state": None if last is None else last.detach()}
    if case["train"]:
        got.update(_grads(s, out, last))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    up = lambda t: None if t is None else t.detach().double().requires_grad_(t.requires_grad)  # noqa: E731
    if case["op"] == "loss":
        x, w = up(s["x"]), up(s["w"])
        rows = torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, w), s["y"], reduction="none")
        if not case["train"]:
            return {"loss": rows.detach()}
        loss = rows.sum() / (s["y"] >= 0).sum()
        dx, dw = torch.autograd.grad(loss, (x, w))
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    q, k, v, g, s0 = (up(s[n]) for n in ("q", "k", "v", "g", "s0"))
    h = case["heads"]
    heads = torch.arange(h, device=DEV) // (h // case["qk_heads"])
    if case["op"] == "step":
        new = torch.exp(g).expand(v.shape[0], h)[:, :, None, None] * s0 + torch.einsum("bhk,bhv->bhkv", k[:, heads], v)
        return {"out": s["scale"] * torch.einsum("bhk,bhkv->bhv", q[:, heads], new), "state": new}
    b, n = case["batch"], case["length"]
    state = torch.zeros(b, h, case["dk"], case["dv"], device=DEV, dtype=torch.float64) if s0 is None else s0
    rate = torch.exp(g).expand(b, n, h)
    outs = []
    for t in range(n):                   # the recurrence, token by token
        new = rate[:, t, :, None, None] * state + k[:, t, heads][..., None] * v[:, t, :, None]
        y = (q[:, t, heads][:, :, None] @ new)[:, :, 0]
        if s["lengths"] is not None:
            live = t < s["lengths"]
            new = torch.where(live[:, None, None, None], new, state)
            y = torch.where(live[:, None, None], y, torch.zeros_like(y))
        state = new
        outs.append(s["scale"] * y)
    out = torch.stack(outs, 1)
    got = {"out": out.detach(), "state": state.detach() if case["state"] else None}
    if case["train"]:
        got.update(_grads(dict(s, q=q, k=k, v=v, g=g, s0=s0, do=s["do"].double(), ds=None if s["ds"] is None else s["ds"].double()), out, state))
    return got
