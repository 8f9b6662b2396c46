"""Linear attention over long sequences: the carried state, and the decay's gradient across the backward's segments.

The reference here is the chunkless definition in float64, summed over the state's tokens at once:
S_t = sum_{s <= t} exp(G_t - G_s) k_s v_s^T + exp(G_t) S_0.
"""
import pytest
import torch

from swiftx_b200 import _lib
from swiftx_b200.linear_attention import linear_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _rand(gen, *s):
    return torch.randn(*s, generator=gen, device=DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L,H", [(4096, 200), (16384, 2)])
def test_the_carried_state_does_not_drift(dtype, L, H):
    """Decays of 1 and a state large against what a chunk adds to it, all of one sign, where whatever an addition cuts off
    adds up.  The state's gradient walks the same way backwards.

    A chunk's sum is added to the state in fp32: one multiply-add, off by half a step, 2^-24 of the state; the sums
    themselves (and the products' 2^-22) are off by (n + 32) 2^-23 of what they add.  Half a step is either sign as
    a rule, but here every chunk adds nearly the same, so all may go the same way: ceil(L / 64) 2^-24 of the
    state.  The segments' chain adds 2 for each segment, at most one for every second chunk.  With products added to the
    state itself in the tensor core it would be 8 additions a chunk of up to 2^-23 each, 16 times the first term."""
    gen = torch.Generator(device=DEV).manual_seed(L)
    dk, dv, scale = 16, 32, 0.25
    pos = lambda *s: (0.5 + torch.rand(*s, generator=gen, device=DEV)).to(dtype)  # noqa: E731
    q, k, v, do = pos(1, L, H, dk), pos(1, L, H, dk), pos(1, L, H, dv), pos(1, L, H, dv)
    # decays of exactly 1; L tokens add about L to a state of 32 L
    g = torch.zeros(1, L, H, device=DEV)
    s0, ds = 32.0 * L * pos(1, H, dk, dv).float(), 32.0 * L * pos(1, H, dk, dv).float()
    x = [t.requires_grad_() for t in (q, k, v, s0)]
    out, state = linear_attention(*x[:3], g, initial_state=s0, scale=scale, return_state=True)
    (ds0,) = torch.autograd.grad([out, state], [s0], [do, ds])
    with torch.no_grad():
        added = torch.einsum("blhk,blhv->bhkv", k.double(), v.double())
        back = scale * torch.einsum("blhk,blhv->bhkv", q.double(), do.double())
        for got, start, sums in ((state, s0, added), (ds0, ds, back)):
            want = start.double() + sums
            chunks = -(-L // 64)
            bound = (2 * chunks + 4) * 2.0 ** -24 * want + (64 + 64) * 2.0 ** -23 * sums
            err = (got.double() - want).abs()
            assert bool((err <= bound).all()), f"largest error over bound {float((err / bound).max()):.3g}"


def _recurrence(q, k, v, g, s0, scale):
    """Token by token, as many heads of q and k as of v."""
    b, L, H, dv = v.shape
    s = torch.zeros(b, H, q.shape[3], dv, device=v.device, dtype=v.dtype) if s0 is None else s0
    a = torch.exp(g).expand(b, L, H)
    outs = []
    for t in range(L):
        s = a[:, t, :, None, None] * s + k[:, t, :, :, None] * v[:, t, :, None]
        outs.append(torch.einsum("bhk,bhkv->bhv", q[:, t], s))
    return scale * torch.stack(outs, 1), s


def _exact(t, do, ds, scale):
    x = {n: v if v is None else v.detach().requires_grad_() for n, v in t.items()}
    out, state = _recurrence(x["q"], x["k"], x["v"], x["g"], x["s0"], scale)
    names = [n for n in x if x[n] is not None]
    outs, dos = ([out, state], [do, ds]) if ds is not None else ([out], [do])
    r = {"d" + n: w for n, w in zip(names, torch.autograd.grad(outs, [x[n] for n in names], dos))}
    return dict(r, out=out.detach(), state=state.detach())


def _case(b, L, H, Hk, dk, dv, dtype, decay, state, flat=1.0):
    """Operands, their float64 forms with q and k repeated for every head, and the upstream gradients."""
    gen = torch.Generator(device=DEV).manual_seed(L + dk)
    g = -flat * torch.rand(*((H,) if decay == "head" else (b, L, H)), generator=gen, device=DEV) ** 4
    t = dict(q=_rand(gen, b, L, Hk, dk).to(dtype), k=_rand(gen, b, L, Hk, dk).to(dtype), v=_rand(gen, b, L, H, dv).to(dtype), g=g,
             s0=_rand(gen, b, H, dk, dv) if state else None)
    do, ds = _rand(gen, b, L, H, dv).to(dtype), _rand(gen, b, H, dk, dv) if state else None
    up = {n: None if x is None else x.double().repeat_interleave(H // Hk, 2) if n in "qk" else x.double() for n, x in t.items()}
    return t, do, ds, up, do.double(), None if ds is None else ds.double()


def _gradients(t, do, ds, scale):
    x = {n: v if v is None else v.detach().requires_grad_() for n, v in t.items()}
    out, state = linear_attention(x["q"], x["k"], x["v"], x["g"], initial_state=x["s0"], scale=scale, return_state=True)
    names = [n for n in x if x[n] is not None]
    outs, dos = ([out, state], [do, ds]) if ds is not None else ([out], [do])
    r = {"d" + n: w for n, w in zip(names, torch.autograd.grad(outs, [x[n] for n in names], dos))}
    return dict(r, out=out.detach(), state=state.detach())


def _segments(b, L, H, dk, dv, dtype):
    a = _lib.LinattnArgs()
    a.batch, a.seqlen, a.heads, a.qk_heads, a.dk, a.dv, a.dtype = b, L, H, 1, dk, dv, 0 if dtype == torch.float32 else 1
    return _lib.load().swx_linattn_segments(a)


def _spread(up, do, ds, scale):
    """Per (row, head): the root of the sum of the squares of the elementary terms of sum_t q_t . dq_t and k_t . dk_t
    (of <S, D> too).  The operator on squared operands, with decays squared, sums the squares."""
    sq = {n: None if x is None else 2 * x if n == "g" else x.square() for n, x in up.items()}
    r = _exact(sq, do.square(), None if ds is None else ds.square(), scale * scale)
    s = (sq["q"] * r["dq"]).sum((1, 3)) + (sq["k"] * r["dk"]).sum((1, 3))
    return (s if sq["s0"] is None else s + (sq["s0"] * r["ds0"]).sum((2, 3))).sqrt()


SEGMENTED = [
    (1, 777, 2, 2, 40, 72, torch.bfloat16, "token", True, 1.0),
    (2, 2100, 3, 3, 40, 72, torch.bfloat16, "token", True, 1.0),       # two slices of v
    (20, 1700, 3, 1, 64, 64, torch.bfloat16, "token", False, 0.05),    # shared q and k, slow decays, a last segment of another length
    (32, 1664, 2, 2, 64, 64, torch.bfloat16, "token", False, 1.0),     # a short last segment: all made shorter
    (1, 4200, 4, 2, 64, 64, torch.bfloat16, "head", True, 1.0),
    (2, 1024, 2, 2, 128, 64, torch.bfloat16, "token", True, 0.05),
    (2, 1500, 3, 3, 40, 56, torch.float32, "token", True, 1.0),
    (1, 2100, 4, 1, 33, 64, torch.float32, "head", True, 0.1),
    (2, 2048, 2, 2, 64, 64, torch.float32, "token", False, 0.05),
]


@pytest.mark.parametrize("b,L,H,Hk,dk,dv,dtype,decay,state,flat", SEGMENTED)
def test_decay_gradient_across_segments(b, L, H, Hk, dk, dv, dtype, decay, state, flat):
    """Each elementary term of dg passes about 16 roundings of at most 2^-23, of either sign: 2^-21 of it, and what the
    tensor cores cut off, always toward zero, as much again: u = 2^-20.  The terms' errors are independent, so they add as
    their squares do: u * _spread for the running sum at each token.  A decay for each head sums the tokens'
    gradients: a term moves those of its segment only (each segment starts from <S, D>), n tokens' the same way, and the m
    segments' errors add as squares: n sqrt(m) u _spread, the rows' as squares too."""
    m = _segments(b, L, H, dk, dv, dtype)
    assert m > 1
    t, do, ds, up, do64, ds64 = _case(b, L, H, Hk, dk, dv, dtype, decay, state, flat)
    got = _gradients(t, do, ds, 0.2)["dg"].double()
    want = _exact(up, do64, ds64, 0.2)["dg"]
    spread = _spread(up, do64, ds64, 0.2)
    if decay == "head":
        bound = 2.0 ** -20 * -(-L // m) * m ** 0.5 * spread.square().sum(0).sqrt()
    else:
        bound = 2.0 ** -20 * spread[:, None].expand(b, L, H)
    err, limit = float((got - want).norm()), float(bound.norm())
    assert err <= limit, f"{err / float(want.norm()):.3g} off, bound {limit / float(want.norm()):.3g}"
    assert limit < 1e-3 * float(want.norm())                  # the bound itself tells something


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("decay", ["token", "head"])
def test_decay_gradient_differences_across_segments(dtype, decay):
    """<dg, direction> against a central difference in float64, h = 1e-6: the difference is off by h^2 of third
    derivatives (up to L^2 times the first, L = 1500: 2^-18 of it) and 2^-52 / h of the sum (below 1e-3).  The
    gradient's errors as above; over a random direction they add as squares, four of that."""
    b, L, H, dk, dv = 1, 1500, 2, 24, 40
    m = _segments(b, L, H, dk, dv, dtype)
    assert m > 1
    t, do, ds, up, do64, ds64 = _case(b, L, H, H, dk, dv, dtype, decay, True)
    got = _gradients(t, do, ds, 0.3)["dg"].double()
    gen = torch.Generator(device=DEV).manual_seed(5)
    d = torch.randn(got.shape, generator=gen, device=DEV, dtype=torch.float64)
    vals = []
    for h in (1e-6, -1e-6):
        out, s = _recurrence(up["q"], up["k"], up["v"], up["g"] + h * d, up["s0"], 0.3)
        vals.append(float((out * do64).sum() + (s * ds64).sum()))
    want = (vals[0] - vals[1]) / 2e-6
    spread = _spread(up, do64, ds64, 0.3)
    bound = -(-L // m) * m ** 0.5 * spread.square().sum(0).sqrt() if decay == "head" else spread[:, None].expand(b, L, H)
    assert abs(float((got * d).sum()) - want) <= 4 * 2.0 ** -20 * float(bound.norm()) + 2.0 ** -18 * abs(want) + 1e-3


@pytest.mark.parametrize("b,L,H,Hk,dk,dv", [(2, 1100, 2, 2, 64, 64), (1, 700, 4, 1, 128, 96), (40, 300, 4, 4, 32, 64), (38, 129, 4, 2, 64, 40),
                                             (19, 250, 8, 8, 48, 64)])
def test_bf16_results_carry_two_roundings(b, L, H, Hk, dk, dv):
    """A result's terms have one factor rounded to bf16 (a score, or the state that is read out), and the result is rounded.
    A rounding of a value of random mantissa is off by 2^-8 / sqrt(3) sqrt(3 / (8 ln 2)) = 1.66e-3 of it in the mean
    square; the terms are of either sign, so a sum's relative error is its terms'.  Two: 2.35e-3; three would be 2.87e-3."""
    t, do, ds, up, do64, ds64 = _case(b, L, H, Hk, dk, dv, torch.bfloat16, "token", True)
    got, want = _gradients(t, do, ds, 0.2), _exact(up, do64, ds64, 0.2)
    for n in ("dq", "dk"):
        want[n] = want[n].unflatten(2, (Hk, H // Hk)).sum(3)
    for n in ("out", "dq", "dk", "dv"):
        err = float((got[n].double() - want[n]).norm() / want[n].norm())
        assert err <= 2.6e-3, (n, err)
