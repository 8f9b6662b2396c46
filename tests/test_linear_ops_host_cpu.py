"""Linear attention and the head's loss on the host: struct layouts, argument checks, plans and workspace sizes of
the C ABI, and the Python layer's refusal of CPU tensors (no GPU needed: every call here returns before a launch)."""
import ctypes

import pytest
import torch

from swiftx_b200 import _lib
from swiftx_b200.linear_attention import linear_attention, linear_attention_step
from swiftx_b200.loss import linear_cross_entropy
from swiftx_b200.sift import SiftConfig, SiftLM

INVALID, UNSUPPORTED = _lib.SWX_ERR_INVALID_ARG, _lib.SWX_ERR_UNSUPPORTED


def _attention(b=2, L=100, H=4, Hk=2, dk=64, dv=64, dtype=1):
    a = _lib.LinattnArgs()
    a.batch, a.seqlen, a.heads, a.qk_heads, a.dk, a.dv, a.dtype = b, L, H, Hk, dk, dv, dtype
    return a


def _xent(T=8, V=100, d=16, dtype=1, reduction=1):
    a = _lib.XentArgs()
    a.tokens, a.vocab, a.dim, a.dtype, a.reduction, a.x_sr, a.w_sr = T, V, d, dtype, reduction, d, d
    a.x = a.weight = 4096
    return a


def test_struct_mirrors_match():
    lib = _lib.load()
    assert lib.swx_xent_args_size() == ctypes.sizeof(_lib.XentArgs)
    assert lib.swx_linattn_args_size() == ctypes.sizeof(_lib.LinattnArgs)


@pytest.mark.parametrize("change,status", [
    (dict(L=-1), INVALID), (dict(b=-1), INVALID), (dict(H=3), INVALID), (dict(Hk=0), INVALID), (dict(dk=0), INVALID),
    (dict(dk=129), UNSUPPORTED), (dict(dv=129), UNSUPPORTED), (dict(dtype=2), UNSUPPORTED), (dict(b=1 << 24, H=1 << 16, Hk=1), UNSUPPORTED),
    (dict(L=1 << 29), UNSUPPORTED), (dict(), INVALID),          # the last: no pointers
])
def test_attention_arguments(change, status):
    lib = _lib.load()
    a = _attention(**change)
    assert lib.swx_linattn_fwd(a, None) == status
    assert lib.swx_linattn_bwd(a, None) == status
    assert lib.swx_linattn_step(a, None) == status
    if change:
        assert lib.swx_linattn_segments(a) == -status
        assert lib.swx_linattn_fwd_workspace_bytes(a) == lib.swx_linattn_bwd_workspace_bytes(a) == -status
    assert lib.swx_linattn_fwd(None, None) == INVALID


def test_attention_plans():
    lib = _lib.load()
    assert lib.swx_linattn_segments(_attention(b=0)) == 1 and lib.swx_linattn_segments(_attention(L=0)) == 1
    assert lib.swx_linattn_fwd(_attention(b=0), None) == _lib.SWX_OK
    assert lib.swx_linattn_segments(_attention(L=64)) == 1                       # one chunk
    for b, L, H, dk, dv in ((1, 65536, 1, 64, 64), (8, 2048, 8, 64, 64), (4, 65536, 32, 64, 64), (1, 4096, 2, 128, 128), (300, 4096, 4, 64, 64)):
        a = _attention(b=b, L=L, H=H, Hk=1, dk=dk, dv=dv)
        n = lib.swx_linattn_segments(a)
        assert 1 <= n <= max(1, L // 128)                                        # at least two chunks each
        assert lib.swx_linattn_bwd_workspace_bytes(a) >= (n > 1) * b * H * n * dk * dv * 4 + 2 * b * H * L * 4


@pytest.mark.parametrize("change,status", [
    (dict(T=-1), INVALID), (dict(V=0), INVALID), (dict(d=0), INVALID), (dict(reduction=3), INVALID), (dict(dtype=2), UNSUPPORTED),
    (dict(T=1 << 29), UNSUPPORTED), (dict(V=1 << 29), UNSUPPORTED), (dict(d=1 << 17), UNSUPPORTED),
])
def test_loss_arguments(change, status):
    lib = _lib.load()
    a = _xent(**change)
    assert lib.swx_xent_fwd(a, None) == status and lib.swx_xent_bwd(a, None) == status
    assert lib.swx_xent_fwd_workspace_bytes(a) == lib.swx_xent_bwd_workspace_bytes(a) == -status
    assert lib.swx_xent_fwd(None, None) == INVALID


def test_loss_buffers():
    lib = _lib.load()
    a = _xent()
    assert lib.swx_xent_fwd(a, None) == INVALID                                   # no outputs
    a.loss = a.count = a.targets = a.row_max = a.row_rsum = a.workspace = 4096
    a.workspace_bytes = lib.swx_xent_fwd_workspace_bytes(a) - 1
    assert lib.swx_xent_fwd(a, None) == INVALID                                   # a short workspace
    a.x_sr = 8
    assert lib.swx_xent_fwd(a, None) == INVALID                                   # rows that overlap
    a.x_sr = 16
    assert lib.swx_xent_bwd(a, None) == _lib.SWX_OK                               # no gradient asked for
    a.dx = 4096
    assert lib.swx_xent_bwd(a, None) == INVALID                                   # no dloss
    a.dloss = 4096
    a.workspace_bytes = lib.swx_xent_bwd_workspace_bytes(a) - 1
    assert lib.swx_xent_bwd(a, None) == INVALID
    a.dweight, a.dw_dtype = 4096, 7
    assert lib.swx_xent_bwd(a, None) == UNSUPPORTED
    f = _xent(dtype=0)
    f.dweight, f.dw_dtype = 4096, 1                                               # fp32 operands, a bf16 gradient
    assert lib.swx_xent_bwd(f, None) == UNSUPPORTED


def test_loss_workspace_off_its_alignment_is_refused():
    lib = _lib.load()
    a = _xent()
    a.loss = a.count = a.targets = a.row_max = a.row_rsum = a.dloss = a.dx = 4096
    a.workspace, a.workspace_bytes = 4096 + 8, 1 << 30
    assert lib.swx_xent_fwd(a, None) == INVALID and lib.swx_xent_bwd(a, None) == INVALID


def test_loss_workspace_does_not_hold_the_logits():
    lib = _lib.load()
    T, V, d = 65536, 131072, 64
    a = _xent(T, V, d)
    logits = 2 * T * V
    assert lib.swx_xent_fwd_workspace_bytes(a) < logits / 16
    assert lib.swx_xent_bwd_workspace_bytes(a) < logits / 16 + 4 * T * d
    b = _xent(T, V, d + 1)                                                        # rows that are not whole 16-byte pieces: copies
    assert lib.swx_xent_bwd_workspace_bytes(b) > lib.swx_xent_bwd_workspace_bytes(a)


def test_cpu_tensors_are_rejected():
    q, v, g = torch.randn(1, 4, 2, 8), torch.randn(1, 4, 2, 8), -torch.rand(1, 4, 2)
    with pytest.raises(RuntimeError):
        linear_attention(q, q, v, g)
    with pytest.raises(RuntimeError):
        linear_attention_step(q[:, 0], q[:, 0], v[:, 0], g[:, 0], torch.zeros(1, 2, 8, 8))
    with pytest.raises(RuntimeError):
        linear_cross_entropy(torch.randn(3, 8), torch.randn(5, 8), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        linear_cross_entropy(torch.randn(3, 8), torch.randn(5, 8), torch.zeros(3, dtype=torch.int64), reduction="max")


def test_model_loss_off_the_gpu_is_forwards_own(monkeypatch):
    """On CPU parameters SiftLM.loss is forward's loss (the mixers are stubbed: they run on CUDA only)."""
    torch.manual_seed(0)
    model = SiftLM(SiftConfig(vocab_size=20, d_model=8, n_layers=1))
    monkeypatch.setattr(type(model.backbone), "forward", lambda self, x: x)
    idx, tgt = torch.randint(0, 20, (2, 5)), torch.randint(0, 20, (2, 5))
    assert torch.equal(model.loss(idx, tgt), model(idx, tgt)[1])
