"""Linear attention (swx_linattn_fwd / _bwd / _step) against the recurrence in float64, token
by token, with gradients from autograd through it.

Tolerances.  Every result is a sum of products; running the same float64 recurrence and
gradients on the absolute values of all inputs gives each result's magnitude sum ``mag``, and a
relative error u in the terms is an error of at most u * mag in the result.
  * bf16 results of bf16 inputs: one rounding of the result (2^-8 of it) and one of a term's
    factor (a score or a state, 2^-8 of the term): 2^-8 (|x| + mag).
  * fp32 results: a term passes n additions in fp32 or in the tensor cores (2^-23 each at most, cut
    off or rounded): per chunk of 64 tokens, 12 products' additions and 2 of the state's update,
    n = 14 ceil(L / 64) + 24, with an exponential (2^-21) and factors kept to 2^-22 or better at
    each of two products: (n + 16) 2^-23 mag; fp32 inputs (three tf32 products, the dropped
    fourth 2^-22): (n + 32) 2^-23 mag, for the products' operands too.
  * the decay's gradient is formed from differences of sums over the sequence: its terms' mag is
    the row's whole sum of |q . dq| + |k . dk|.
"""
import pytest
import torch

from swiftx_b200 import _lib
from swiftx_b200.linear_attention import linear_attention, linear_attention_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAMES = ("q", "k", "v", "g", "s0")


def _inputs(b, L, H, Hk, dk, dv, dtype, decay="token", state=True, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    g = -torch.rand(*((H,) if decay == "head" else (b, L, H)), generator=gen, device=DEV) ** 4
    t = dict(q=rand(b, L, Hk, dk).to(dtype), k=rand(b, L, Hk, dk).to(dtype), v=rand(b, L, H, dv).to(dtype), g=g,
             s0=rand(b, H, dk, dv) if state else None)
    return t, rand(b, L, H, dv).to(dtype), rand(b, H, dk, dv) if state else None


def _recurrence(q, k, v, g, s0, scale, lengths):
    b, L, H, dv = v.shape
    heads = torch.arange(H, device=v.device) // (H // q.shape[2])
    s = torch.zeros(b, H, q.shape[3], dv, device=v.device, dtype=v.dtype) if s0 is None else s0
    a = torch.exp(g).expand(b, L, H)
    outs = []
    for t in range(L):
        new = a[:, t, :, None, None] * s + k[:, t, heads][..., None] * v[:, t, :, None]
        y = torch.einsum("bhk,bhkv->bhv", q[:, t, heads], new)
        if lengths is not None:
            live = t < lengths
            new = torch.where(live[:, None, None, None], new, s)
            y = torch.where(live[:, None, None], y, torch.zeros_like(y))
        s = new
        outs.append(y)
    return (scale * torch.stack(outs, 1) if outs else torch.zeros_like(v)), s


def _oracle(t, do, ds, scale, lengths, absolute=False):
    """out, state and every gradient in float64 (of the inputs' absolute values when asked)."""
    up = lambda x: None if x is None else (x.detach().double().abs() if absolute else x.detach().double())  # noqa: E731
    x = {n: (t[n].detach().double() if n == "g" else up(t[n])) for n in NAMES}
    x = {n: None if v is None else v.requires_grad_() for n, v in x.items()}
    out, state = _recurrence(*(x[n] for n in NAMES), scale, lengths)
    r = {"out": out.detach(), "state": state.detach()}
    if do is not None:
        names = [n for n in NAMES if x[n] is not None]
        outs, dos = [out], [up(do)]
        if ds is not None:
            outs, dos = outs + [state], dos + [up(ds)]
        r.update({"d" + n: w for n, w in zip(names, torch.autograd.grad(outs, [x[n] for n in names], dos))})
    return r


def _run(t, do, ds, scale, lengths):
    x = {n: None if v is None else v.detach().requires_grad_() for n, v in t.items()}
    out, state = linear_attention(x["q"], x["k"], x["v"], x["g"], initial_state=x["s0"], scale=scale, lengths=lengths,
                                  return_state=True)
    names = [n for n in NAMES if x[n] is not None]
    outs, dos = ([out, state], [do, ds]) if ds is not None else ([out], [do])
    r = {"out": out.detach(), "state": state.detach()}
    r.update({"d" + n: w for n, w in zip(names, torch.autograd.grad(outs, [x[n] for n in names], dos))})
    return r


def _check(got, want, mag, t, L):
    dtype = t["v"].dtype
    n = 14 * -(-L // 64) + 24
    u = (n + (32 if dtype == torch.float32 else 16)) * 2.0 ** -23
    m = dict(mag)
    if "dg" in mag:
        # per (row, head): the whole sum of |q . dq| + |k . dk|, of the heads that share q and k together
        H, Hk = t["v"].shape[2], t["q"].shape[2]
        mass = sum((t[a].double().abs() * mag["d" + a]).sum((1, 3)) for a in "qk").repeat_interleave(H // Hk, 1)
        mass = mass + (t["s0"].double().abs() * mag["ds0"]).sum((2, 3)) if t["s0"] is not None else mass
        m["dg"] = mass.sum(0) if mag["dg"].dim() == 1 else mass[:, None].expand_as(mag["dg"])
    for name, w in want.items():
        x = got[name]
        bound = u * m[name]
        if x.dtype == torch.bfloat16:
            bound = 1.02 * 2.0 ** -8 * (w.abs() + m[name]) + bound
        err = (x.double() - w).abs()
        assert x.shape == w.shape and bool((err <= bound + 1e-30).all()), \
            f"{name}: largest error over bound {float((err / (bound + 1e-30)).max()):.3g}"


SHAPES = [
    # b, L, H, Hk, dk, dv, dtype, decay, state
    (2, 1, 2, 2, 64, 64, torch.bfloat16, "token", True),       # one token
    (1, 63, 3, 3, 64, 64, torch.bfloat16, "token", False),     # a chunk less one
    (2, 64, 2, 1, 32, 16, torch.bfloat16, "head", True),       # one chunk, shared heads
    (1, 65, 2, 2, 64, 64, torch.float32, "token", True),       # a chunk and one
    (2, 300, 4, 2, 40, 56, torch.float32, "token", True),      # odd head sizes, segments
    (1, 777, 2, 2, 64, 128, torch.bfloat16, "token", True),    # two slices of v
    (2, 200, 3, 1, 128, 65, torch.bfloat16, "head", False),    # a wide state, a slice of one column
    (3, 130, 6, 2, 1, 1, torch.bfloat16, "token", True),       # scalar states
    (1, 513, 2, 2, 127, 33, torch.float32, "head", True),      # rows that are not whole 16-byte pieces
    (1, 1100, 1, 1, 16, 64, torch.bfloat16, "token", True),    # many segments of one head
]


@pytest.mark.parametrize("b,L,H,Hk,dk,dv,dtype,decay,state", SHAPES)
def test_forward_and_gradients(b, L, H, Hk, dk, dv, dtype, decay, state):
    t, do, ds = _inputs(b, L, H, Hk, dk, dv, dtype, decay, state, seed=L + dk)
    scale = dk ** -0.5
    got = _run(t, do, ds, scale, None)
    _check(got, _oracle(t, do, ds, scale, None), _oracle(t, do, ds, scale, None, True), t, L)


@pytest.mark.parametrize("b,L,H,Hk,dk,dv,decay,state", [
    (16, 520, 8, 8, 64, 64, "token", False),       # five chunks of 128, the last with 8 tokens; one walk a head
    (3, 2100, 6, 3, 40, 72, "token", True),        # a slice of 8 columns, shared heads, four segments
    (1, 4200, 8, 2, 64, 64, "head", True),         # eight segments; the backward's are others
    (20, 1030, 8, 1, 24, 64, "token", True),       # more heads than SMs
])
def test_pipelined_kernels(b, L, H, Hk, dk, dv, decay, state):
    """Sizes that the pipelined bf16 kernels take (chunks of 128 tokens, a ring of three)."""
    t, do, ds = _inputs(b, L, H, Hk, dk, dv, torch.bfloat16, decay, state, seed=L)
    got = _run(t, do, ds, 0.2, None)
    _check(got, _oracle(t, do, ds, 0.2, None), _oracle(t, do, ds, 0.2, None, True), t, L)
    assert _lib.load().swx_device_wait_status() == _lib.SWX_OK
    with torch.no_grad():                          # without the backward's states: the same values
        out, last = linear_attention(t["q"], t["k"], t["v"], t["g"], initial_state=t["s0"], scale=0.2, return_state=True)
    assert torch.equal(out, got["out"]) and torch.equal(last, got["state"])


@pytest.mark.parametrize("b,L,H,dk,dv,odd", [
    (1, 1100, 2, 64, 64, True), (3, 700, 2, 33, 72, True),        # cut into segments
    (40, 200, 4, 32, 32, False), (2, 64, 3, 64, 64, False),       # many heads, a single short chunk
])
def test_bf16_kernels_of_short_chunks(b, L, H, dk, dv, odd):
    """bf16 calls that the pipelined kernels do not take: tensors off 16-byte borders, and sizes."""
    t, do, ds = _inputs(b, L, H, H, dk, dv, torch.bfloat16, seed=L + H)
    if odd:
        t = {n: torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape) for n, x in t.items()}
    got = _run(t, do, ds, 0.2, None)
    _check(got, _oracle(t, do, ds, 0.2, None), _oracle(t, do, ds, 0.2, None, True), t, L)


def test_pipelined_padded_steep_and_reset_rows():
    """Lengths on and off the chunks' borders with NaN behind them; resets, decays too steep for the split
    exponentials (2^-60 inside 16 tokens), and decays of 0, in the pipelined kernels."""
    b, L, H, dk, dv = 8, 700, 16, 64, 64
    t, do, ds = _inputs(b, L, H, H, dk, dv, torch.bfloat16, seed=17)
    t["g"][0, 130, :8] = -float("inf")
    t["g"][1, :, 3] = -30.0
    t["g"][2] = 0.0
    t["g"][3, 200:260, 5] = -200.0
    n = torch.tensor([700, 0, 1, 128, 129, 640, 699, 5000], device=DEV)
    got = _run(t, do, ds, 0.125, n)
    _check(got, _oracle(t, do, ds, 0.125, n), _oracle(t, do, ds, 0.125, n, True), t, L)
    behind = torch.arange(L, device=DEV)[None, :] >= n[:, None]
    for k in ("q", "k", "v", "g"):
        t[k][behind] = float("nan")
    dirty = _run(t, do, ds, 0.125, n)
    for k in got:
        assert torch.equal(got[k], dirty[k]), k
    assert torch.count_nonzero(got["out"][behind]) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths", [[0, 1, 64, 65], [200, 199, 5, 130], [-3, 1000, 128, 0]])
def test_padded_rows(dtype, lengths):
    """Each row ends at its own length; NaN behind it changes nothing; zeros there in every result."""
    b, L = 4, 200
    t, do, ds = _inputs(b, L, 2, 2, 48, 72, dtype, seed=7)
    n = torch.tensor(lengths, device=DEV)
    clean = _run(t, do, ds, 0.25, n)
    _check(clean, _oracle(t, do, ds, 0.25, n), _oracle(t, do, ds, 0.25, n, True), t, L)
    behind = torch.arange(L, device=DEV)[None, :] >= n[:, None]
    bad = {k: v.clone() for k, v in t.items()}
    for k in ("q", "k", "v", "g"):
        bad[k][behind] = float("nan")
    do = do.clone()
    do[behind] = float("inf")
    dirty = _run(bad, do, ds, 0.25, n)
    for k in clean:
        assert torch.equal(clean[k], dirty[k]), k
    for k in ("out", "dq", "dk", "dv", "dg"):
        assert torch.count_nonzero(clean[k][behind]) == 0, k
    assert torch.equal(clean["state"][n <= 0], t["s0"][n <= 0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_resets_and_extreme_decays(dtype):
    """-inf (and the type's lowest value) forget everything before; 0 keeps it; -200 a token underflows."""
    b, L, H = 1, 190, 4
    t, do, ds = _inputs(b, L, H, H, 32, 32, dtype, seed=3)
    t["g"][:, 70, 0] = -float("inf")
    t["g"][:, 128, 0] = torch.finfo(torch.float32).min
    t["g"][..., 1] = 0.0
    t["g"][..., 2] = -200.0
    t["g"][:, :, 3] = -float("inf")
    got = _run(t, do, ds, 0.5, None)
    _check(got, _oracle(t, do, ds, 0.5, None), _oracle(t, do, ds, 0.5, None, True), t, L)
    assert torch.count_nonzero(got["dg"][:, :, 3]) == 0 and float(got["dg"][0, 70, 0]) == 0.0
    # nothing before the reset reaches behind it
    other = {k: v.clone() for k, v in t.items()}
    for k in "qkv":
        other[k][:, :70] = 3.0
    other["s0"] += 5.0
    again = _run(other, do, ds, 0.5, None)
    assert torch.equal(again["out"][:, 70:, 0], got["out"][:, 70:, 0])


@pytest.mark.parametrize("b,L,H,dtype", [(1, 190, 4, torch.bfloat16), (2, 190, 4, torch.float32), (32, 520, 4, torch.bfloat16)])
def test_growing_states(b, L, H, dtype):
    """Positive log decays: sums that swing by 4 either way, a rise and fall by 36 inside 24 tokens, and one by 50 in
    20 (beyond what the pipelined kernel's split exponentials take).  The terms' errors are as with decays below 0."""
    t, do, ds = _inputs(b, L, H, H, 32, 40, dtype, seed=4)
    at = torch.arange(L, device=DEV)
    t["g"][..., 0] = 0.4 * torch.cos(at * (2 * torch.pi / 64))
    t["g"][..., 1] += 0.01
    t["g"][:, 100:112, 2], t["g"][:, 112:124, 2] = 3.0, -3.0
    t["g"][:, 130:140, 3], t["g"][:, 140:150, 3] = 5.0, -5.0
    got = _run(t, do, ds, 0.2, None)
    _check(got, _oracle(t, do, ds, 0.2, None), _oracle(t, do, ds, 0.2, None, True), t, L)


def test_strided_operands():
    """Column slices of one projection's output, a transposed head layout, a broadcast decay and gradient."""
    b, L, H, d = 2, 150, 4, 64
    gen = torch.Generator(device=DEV).manual_seed(5)
    qkv = torch.randn(b, L, 3 * H * d + 8, generator=gen, device=DEV).to(torch.bfloat16)
    q, k, v = (qkv[..., 8 + i * H * d:8 + (i + 1) * H * d].unflatten(-1, (H, d)) for i in range(3))
    k = k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    g = -torch.rand(H, generator=gen, device=DEV)
    t = dict(q=q, k=k, v=v, g=g[None, None].expand(b, L, H), s0=None)
    do = torch.randn(1, 1, H, d, generator=gen, device=DEV).to(torch.bfloat16).expand(b, L, H, d)
    got = _run(t, do, None, 0.125, None)
    _check(got, _oracle(t, do, None, 0.125, None), _oracle(t, do, None, 0.125, None, True), t, L)
    # A last dimension that is not contiguous gives the same values through copies.  Odd offsets keep TMA away: the
    # kernels with chunks of 64 tokens, whose sums round at other places than those with chunks of 128 (both are within the
    # bound of the exact values, so they may differ by up to twice it).
    dense = _run({n: None if x is None else x.contiguous() for n, x in t.items()}, do.contiguous(), None, 0.125, None)
    odd = {n: None if x is None else torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape) for n, x in t.items()}
    swapped = {n: x if n in ("g", "s0") else x.transpose(-1, -2).contiguous().transpose(-1, -2) for n, x in t.items()}
    _check(_run(odd, do, None, 0.125, None), _oracle(t, do, None, 0.125, None), _oracle(t, do, None, 0.125, None, True), t, L)
    other = _run(swapped, do, None, 0.125, None)
    for name in dense:
        assert torch.equal(dense[name], other[name]), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_directional_differences(dtype):
    """<gradient, direction> against a central difference of the float64 recurrence: the difference's own
    error is O(h^2) (h = 1e-4 in float64: 1e-8 of third derivatives of order 1e2)."""
    t, do, ds = _inputs(2, 140, 2, 1, 24, 40, dtype, seed=11)
    got = _run(t, do, ds, 0.3, None)
    gen = torch.Generator(device=DEV).manual_seed(12)
    for name in NAMES:
        d = torch.randn(t[name].shape, generator=gen, device=DEV, dtype=torch.float64)
        vals = []
        for h in (1e-4, -1e-4):
            x = {n: v.double() for n, v in t.items()}
            x[name] = x[name] + h * d
            out, s = _recurrence(*(x[n] for n in NAMES), 0.3, None)
            vals.append(float((out * do.double()).sum() + (s * ds.double()).sum()))
        want = (vals[0] - vals[1]) / 2e-4
        have = float((got["d" + name].double() * d).sum())
        # each gradient value carries at most twice a bf16 rounding (or 2^-14 of it in fp32); over a
        # random direction the errors add as their squares do; eight of that
        eps = 2.0 ** -7 if got["d" + name].dtype == torch.bfloat16 else 2.0 ** -14
        assert abs(have - want) <= 8 * eps * float(got["d" + name].double().norm()) + 1e-3, name


def test_partial_gradients_and_outputs():
    """A gradient of the state alone, an unused output, operands that want none."""
    t, do, ds = _inputs(1, 100, 2, 2, 32, 32, torch.float32, seed=2)
    x = {n: v.detach().requires_grad_(n in ("k", "s0")) for n, v in t.items()}
    out, state = linear_attention(x["q"], x["k"], x["v"], x["g"], initial_state=x["s0"], return_state=True)
    dk, ds0 = torch.autograd.grad(state, (x["k"], x["s0"]), ds)
    want = _oracle(t, torch.zeros_like(do), ds, 1.0, None)
    mag = _oracle(t, torch.zeros_like(do), ds, 1.0, None, True)
    for got, name in ((dk, "dk"), (ds0, "ds0")):
        assert bool(((got.double() - want[name]).abs() <= 100 * 2.0 ** -23 * mag[name] + 1e-30).all())
    with torch.no_grad():
        alone = linear_attention(x["q"], x["k"], x["v"], x["g"], initial_state=x["s0"])
    assert torch.equal(alone, out.detach()) and not alone.requires_grad


def test_deterministic_and_other_streams():
    t, do, ds = _inputs(2, 700, 3, 1, 64, 96, torch.bfloat16, seed=1)
    a = _run(t, do, ds, 0.1, None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _run(t, do, ds, 0.1, None)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_empty():
    for b, L in ((0, 5), (3, 0)):
        t, do, ds = _inputs(b, L, 2, 1, 16, 24, torch.float32, "head", True)
        r = _run(t, do, ds, 1.0, None)
        assert r["out"].shape == (b, L, 2, 24) and torch.equal(r["state"], t["s0"]) and torch.equal(r["ds0"], ds)
        assert torch.count_nonzero(r["dg"]) == 0
    out, state = linear_attention(t["q"], t["k"], t["v"], t["g"], return_state=True)
    assert torch.count_nonzero(state) == 0


@pytest.mark.parametrize("b,H,Hk,dk,dv,dtype,decay", [
    (1, 8, 8, 64, 64, torch.float32, "token"),
    (5, 6, 2, 128, 128, torch.bfloat16, "head"),
    (3, 2, 1, 1, 1, torch.bfloat16, "token"),
    (2, 4, 4, 37, 129 - 64, torch.float32, "token"),
    (33, 3, 3, 16, 36, torch.bfloat16, "token"),
])
def test_step(b, H, Hk, dk, dv, dtype, decay):
    """fp32 arithmetic: a product and an addition in the state's update (and the exponential, 2 ulp),
    dk additions in the readout; bf16 results one rounding more."""
    t, _, _ = _inputs(b, 1, H, Hk, dk, dv, dtype, decay, True, seed=b)
    args = [t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], t["g"] if decay == "head" else t["g"][:, 0]]
    want, mag = _oracle(t, None, None, 0.3, None), _oracle(t, None, None, 0.3, None, True)
    state = t["s0"].clone()
    out = linear_attention_step(*args, state, scale=0.3)
    assert bool(((state.double() - want["state"]).abs() <= 5 * 2.0 ** -24 * mag["state"]).all())
    bound = (dk + 8) * 2.0 ** -24 * mag["out"][:, 0]
    if dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * want["out"][:, 0].abs()
    assert out.dtype == dtype and bool(((out.double() - want["out"][:, 0]).abs() <= bound * 1.01).all())
    # strided rows
    wide = torch.zeros(b, 2 * Hk, dk + 3, device=DEV, dtype=dtype)
    wide[:, ::2, 1:dk + 1] = args[0]
    again = t["s0"].clone()
    assert torch.equal(linear_attention_step(wide[:, ::2, 1:dk + 1], *args[1:], again, scale=0.3), out)
    assert torch.equal(again, state)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_then_tokens(dtype):
    """A prompt in two pieces and single tokens behind it give what one long call gives: out within both
    calls' bounds, the state within twice the sequence bound."""
    L, cut, tail = 230, 100, 6
    t, _, _ = _inputs(2, L, 4, 2, 64, 64, dtype, seed=9)
    part = lambda a, b: [t[n][:, a:b] for n in ("q", "k", "v", "g")]  # noqa: E731
    whole, last = linear_attention(*part(0, L), initial_state=t["s0"], scale=0.125, return_state=True)
    o1, s1 = linear_attention(*part(0, cut), initial_state=t["s0"], scale=0.125, return_state=True)
    o2, s2 = linear_attention(*part(cut, L - tail), initial_state=s1, scale=0.125, return_state=True)
    steps = [linear_attention_step(*(t[n][:, i] for n in ("q", "k", "v", "g")), s2, scale=0.125) for i in range(L - tail, L)]
    got = torch.cat([o1, o2, torch.stack(steps, 1)], 1)
    mag = _oracle(t, None, None, 0.125, None, True)
    u = 2 * (14 * 4 + 24 + 32) * 2.0 ** -23
    assert bool(((s2 - last).double().abs() <= u * mag["state"]).all())
    ub = u + (3 * 1.02 * 2.0 ** -8 if dtype == torch.bfloat16 else 0)
    assert bool(((got - whole).double().abs() <= ub * mag["out"]).all())


def test_captured_calls():
    """Forward, backward and step captured into two graphs that live side by side and are replayed with new values."""
    def build(seed):
        t, do, ds = _inputs(1, 400, 2, 2, 64, 64, torch.bfloat16, seed=seed)
        t = {n: v.clone().requires_grad_() for n, v in t.items()}
        state = torch.zeros(1, 2, 64, 64, device=DEV)

        def f():
            out, s = linear_attention(t["q"], t["k"], t["v"], t["g"], initial_state=t["s0"], return_state=True)
            grads = torch.autograd.grad([out, s], [t[n] for n in NAMES], [do, ds])
            with torch.no_grad():
                y = linear_attention_step(t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], t["g"][:, 0], state)
            return [out.detach(), s.detach(), *grads, y]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        state.zero_()
        with torch.cuda.graph(graph):
            r = f()
        return t, state, f, graph, r

    runs = [build(21), build(22)]
    for t, state, f, graph, r in runs:
        with torch.no_grad():
            for n in "qkv":
                t[n].mul_(0.5)
    for t, state, f, graph, r in runs:
        state.zero_()
        graph.replay()
    torch.cuda.synchronize()
    for t, state, f, graph, r in runs:
        kept = [x.clone() for x in r]
        state.zero_()
        for a, b in zip(kept, f()):
            assert torch.equal(a, b)


def test_refusals():
    t, _, _ = _inputs(2, 10, 4, 2, 16, 16, torch.bfloat16)
    q, k, v, g, s0 = (t[n] for n in NAMES)
    bad = [
        dict(q=q[0]), dict(k=k[:, :5]), dict(q=q.float()), dict(q=q.double(), k=k.double(), v=v.double()),
        dict(g=g.bfloat16()), dict(g=g[:, :, :2]), dict(g=g[:1]), dict(s0=s0.bfloat16()), dict(s0=s0[:1]),
        dict(v=v[:, :, :3], g=g[:, :, :3], s0=s0[:, :3]),
        dict(q=torch.zeros(2, 10, 2, 129, device=DEV).bfloat16(), k=torch.zeros(2, 10, 2, 129, device=DEV).bfloat16(), s0=None),
        dict(v=torch.zeros(2, 10, 4, 0, device=DEV).bfloat16(), s0=None),
    ]
    for change in bad:
        x = dict(t, **change)
        with pytest.raises(ValueError):
            linear_attention(x["q"], x["k"], x["v"], x["g"], initial_state=x["s0"])
    for lengths in (torch.tensor([1, 2]), torch.tensor([1, 2], device=DEV, dtype=torch.int32), torch.tensor([1], device=DEV)):
        with pytest.raises(ValueError):
            linear_attention(q, k, v, g, lengths=lengths)
    with pytest.raises(RuntimeError):
        linear_attention(q.cpu(), k.cpu(), v.cpu(), g.cpu())
    one = [x[:, 0] for x in (q, k, v, g)]
    with pytest.raises(ValueError):
        linear_attention_step(*one, s0.transpose(-1, -2).contiguous().transpose(-1, -2))
    with pytest.raises(ValueError):
        linear_attention_step(q, k, v, g, s0)
    x = q.detach().float().requires_grad_()
    y = linear_attention(x, k.float(), v.float(), g)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):                  # no second derivatives
        dx.sum().backward()


def test_short_buffers_are_refused_on_the_host():
    lib = _lib.load()
    t, do, _ = _inputs(1, 1000, 2, 2, 64, 64, torch.bfloat16, state=False)
    a = _lib.LinattnArgs()
    a.batch, a.seqlen, a.heads, a.qk_heads, a.dk, a.dv, a.dtype = 1, 1000, 2, 2, 64, 64, 1
    a.q = a.k = t["q"].data_ptr()
    a.v, a.log_decay, a.out = t["v"].data_ptr(), t["g"].data_ptr(), t["v"].data_ptr()
    assert lib.swx_linattn_segments(a) > 1 and lib.swx_linattn_fwd_workspace_bytes(a) > 0
    assert lib.swx_linattn_fwd(a, None) == _lib.SWX_ERR_INVALID_ARG            # no workspace
    a.seg_states = a.workspace = t["g"].data_ptr()
    a.workspace_bytes = lib.swx_linattn_fwd_workspace_bytes(a) - 4
    assert lib.swx_linattn_fwd(a, None) == _lib.SWX_ERR_INVALID_ARG
    a.dout = a.dq = a.dk_out = a.dv_out = t["q"].data_ptr()
    a.dlog_decay = t["g"].data_ptr()
    a.workspace_bytes = lib.swx_linattn_bwd_workspace_bytes(a) - 4
    assert lib.swx_linattn_bwd(a, None) == _lib.SWX_ERR_INVALID_ARG


def test_step_and_autograd():
    """A step takes no operand that a gradient is asked of, and a backward that saved the state before it raises."""
    t, do, _ = _inputs(1, 3, 2, 2, 16, 16, torch.float32)
    one = [t[n][:, 0] for n in ("q", "k", "v", "g")]
    for i in range(5):
        x = [*one, t["s0"].clone()]
        x[i] = x[i].detach().requires_grad_()
        with pytest.raises(RuntimeError, match="not differentiable"):
            linear_attention_step(*x)
        with torch.no_grad():
            linear_attention_step(*x)
    q = t["q"].detach().requires_grad_()
    state = t["s0"].clone()
    out = linear_attention(q, t["k"], t["v"], t["g"], initial_state=state)
    linear_attention_step(*one, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(do)
