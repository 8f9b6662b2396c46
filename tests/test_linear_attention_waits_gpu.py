"""The pipelined linear-attention kernels when a wait runs out: they stop issuing copies and products, see those under
way end, record the timeout and return; the next call is unharmed.

No failure is provoked: with wait_polls below 0 every wait of the kernels' roles for one another gives up at once,
while the copies already issued are still waited for (with the default limit)."""
import pytest
import torch

from swiftx_b200 import _lib
from swiftx_b200.linear_attention import _args, linear_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("b,L,H,cut", [(2, 640, 4, False), (1, 4096, 40, True)])
def test_waits_that_give_up(b, L, H, cut):
    """More chunks than the ring has places, in one walk and in segments (the state kernel too)."""
    lib = _lib.load()
    gen = torch.Generator(device=DEV).manual_seed(L)
    q, k, v = (torch.randn(b, L, H, 64, generator=gen, device=DEV).to(torch.bfloat16) for _ in range(3))
    g = -torch.rand(b, L, H, generator=gen, device=DEV)
    before = linear_attention(q, k, v, g, return_state=True)
    assert lib.swx_device_wait_status() == _lib.SWX_OK
    a = _args(q, k, v, g, 1.0)
    n = lib.swx_linattn_fwd_workspace_bytes(a)
    assert (n > 0) == cut
    out, last, ws = torch.empty_like(v), g.new_empty(b, H, 64, 64), g.new_empty(n // 4 + 4)
    a.out, a.final_state, a.workspace, a.workspace_bytes = out.data_ptr(), last.data_ptr(), ws.data_ptr(), n
    a.wait_polls = -1
    assert lib.swx_linattn_fwd(a, _lib.stream_ptr(q.device)) == _lib.SWX_OK
    assert lib.swx_device_wait_status() == _lib.SWX_ERR_TIMEOUT
    a.wait_polls = 1 << 16
    assert lib.swx_linattn_fwd(a, _lib.stream_ptr(q.device)) == _lib.SWX_OK
    assert lib.swx_device_wait_status() == _lib.SWX_OK
    assert torch.equal(out, before[0]) and torch.equal(last, before[1])
    for x, y in zip(linear_attention(q, k, v, g, return_state=True), before):
        assert torch.equal(x, y)
