"""Linear attention over long sequences: the carried state against its definition in float64."""
import pytest
import torch

from swiftx_b200.linear_attention import linear_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


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
