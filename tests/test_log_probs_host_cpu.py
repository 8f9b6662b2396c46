"""Scoring and distillation on the host: struct layouts, argument checks and workspace sizes of the C ABI, and the Python
layer's refusal of CPU tensors (no GPU needed: every call here returns before a launch)."""
import ctypes

import pytest
import torch

from swiftx_b200 import _lib
from swiftx_b200.log_probs import linear_log_probs, token_log_probs
from swiftx_b200.loss import linear_distillation
from swiftx_b200.sift import SiftConfig, SiftLM

INVALID, UNSUPPORTED = _lib.SWX_ERR_INVALID_ARG, _lib.SWX_ERR_UNSUPPORTED


def _score(T=8, V=100, d=16, dtype=1, top=0, temp=1.0):
    a = _lib.LogprobArgs()
    a.tokens, a.vocab, a.dim, a.dtype, a.top_k, a.temperature, a.x_sr, a.w_sr = T, V, d, dtype, top, temp, d, d
    a.x = a.weight = 4096
    return a


def _distill(T=8, V=100, d=16, dtype=1, K=4, temp=1.0, reduction=1, teacher=0):
    a = _lib.DistillArgs()
    a.tokens, a.vocab, a.dim, a.dtype, a.entries, a.temperature, a.x_sr, a.w_sr = T, V, d, dtype, K, temp, d, d
    a.reduction, a.teacher_dtype, a.ids_sr, a.tl_sr = reduction, teacher, K, K
    a.x = a.weight = 4096
    return a


def test_struct_mirrors_match():
    lib = _lib.load()
    assert lib.swx_logprob_args_size() == ctypes.sizeof(_lib.LogprobArgs)
    assert lib.swx_distill_args_size() == ctypes.sizeof(_lib.DistillArgs)


_SIZES = [(dict(T=-1), INVALID), (dict(V=0), INVALID), (dict(d=0), INVALID), (dict(dtype=2), UNSUPPORTED), (dict(T=1 << 29), UNSUPPORTED),
          (dict(V=1 << 29), UNSUPPORTED), (dict(d=1 << 17), UNSUPPORTED), (dict(temp=0.0), INVALID), (dict(temp=-1.0), INVALID),
          (dict(temp=float("nan")), INVALID), (dict(temp=float("inf")), INVALID)]


@pytest.mark.parametrize("change,status", _SIZES + [(dict(top=-1), INVALID), (dict(top=101), INVALID), (dict(V=1000, top=129), UNSUPPORTED)])
def test_scoring_arguments(change, status):
    lib = _lib.load()
    a = _score(**change)
    assert lib.swx_logprob_fwd(a, None) == status and lib.swx_logprob_bwd(a, None) == status
    assert lib.swx_logprob_fwd_workspace_bytes(a) == lib.swx_logprob_bwd_workspace_bytes(a) == -status
    if "d" not in change:
        assert lib.swx_token_logprob(a, None) == status
    assert lib.swx_logprob_fwd(None, None) == lib.swx_logprob_bwd(None, None) == lib.swx_token_logprob(None, None) == INVALID


@pytest.mark.parametrize("change,status", _SIZES + [(dict(K=0), INVALID), (dict(K=129), UNSUPPORTED), (dict(reduction=3), INVALID),
                                                     (dict(teacher=2), UNSUPPORTED)])
def test_distillation_arguments(change, status):
    lib = _lib.load()
    a = _distill(**change)
    assert lib.swx_distill_fwd(a, None) == status and lib.swx_distill_bwd(a, None) == status
    assert lib.swx_distill_fwd_workspace_bytes(a) == lib.swx_distill_bwd_workspace_bytes(a) == lib.swx_distill_saved_bytes(a) == -status
    assert lib.swx_distill_fwd(None, None) == lib.swx_distill_bwd(None, None) == INVALID


def test_scoring_buffers():
    lib = _lib.load()
    a = _score(top=3)
    assert lib.swx_logprob_fwd(a, None) == INVALID                               # no outputs
    a.targets = a.log_probs = a.entropy = a.top_log_probs = a.top_ids = a.workspace = 4096
    a.workspace_bytes = lib.swx_logprob_fwd_workspace_bytes(a) - 1
    assert lib.swx_logprob_fwd(a, None) == INVALID                               # a short workspace
    a.workspace_bytes, a.row_max = 1 << 30, 4096
    assert lib.swx_logprob_fwd(a, None) == INVALID                               # one of the two statistics
    a.row_sum, a.workspace = 4096, 4096 + 8
    assert lib.swx_logprob_fwd(a, None) == INVALID                               # a workspace off 16 bytes
    a.workspace, a.top_ids = 4096, None
    assert lib.swx_logprob_fwd(a, None) == INVALID                               # alternatives without their ids
    a.x_sr = 8
    assert lib.swx_logprob_fwd(a, None) == INVALID                               # rows that overlap
    a.x_sr = 16
    assert lib.swx_logprob_bwd(a, None) == _lib.SWX_OK                           # no gradient asked for
    a.dx, a.workspace_bytes = 4096, lib.swx_logprob_bwd_workspace_bytes(a) - 1
    assert lib.swx_logprob_bwd(a, None) == INVALID
    a.workspace_bytes, a.entropy, a.d_entropy = 1 << 30, None, 4096
    assert lib.swx_logprob_bwd(a, None) == INVALID                               # the entropy's gradient without the entropy
    a.dweight, a.dw_dtype = 4096, 7
    assert lib.swx_logprob_bwd(a, None) == UNSUPPORTED
    b = _score()
    assert lib.swx_token_logprob(b, None) == INVALID                             # no output
    b.entropy, b.targets = 4096, 4096
    assert lib.swx_token_logprob(b, None) == INVALID                             # targets without a place for their values


def test_distillation_buffers():
    lib = _lib.load()
    a = _distill()
    assert lib.swx_distill_fwd(a, None) == INVALID
    a.loss = a.count = a.teacher_ids = a.teacher_logits = a.saved = a.workspace = 4096
    a.saved_bytes = lib.swx_distill_saved_bytes(a)
    a.workspace_bytes = lib.swx_distill_fwd_workspace_bytes(a) - 1
    assert lib.swx_distill_fwd(a, None) == INVALID                               # a short workspace
    a.workspace_bytes, a.workspace = 1 << 30, 4096 + 8
    assert lib.swx_distill_fwd(a, None) == INVALID                               # off 16 bytes
    a.workspace, a.saved_bytes = 4096, a.saved_bytes - 1
    assert lib.swx_distill_fwd(a, None) == INVALID                               # too little to keep for the backward
    a.saved_bytes, a.saved = 1 << 30, 4096 + 8
    assert lib.swx_distill_fwd(a, None) == INVALID
    a.saved = 4096
    assert lib.swx_distill_bwd(a, None) == _lib.SWX_OK                           # no gradient asked for
    a.dx = 4096
    assert lib.swx_distill_bwd(a, None) == INVALID                               # no dloss
    a.dloss, a.workspace_bytes = 4096, lib.swx_distill_bwd_workspace_bytes(a) - 1
    assert lib.swx_distill_bwd(a, None) == INVALID
    f = _distill(dtype=0)
    f.dweight, f.dw_dtype = 4096, 1                                              # fp32 operands, a bf16 gradient
    assert lib.swx_distill_bwd(f, None) == UNSUPPORTED


def test_workspaces_do_not_hold_the_logits():
    """Scoring takes 8192 rows at a time: statistics of 16 bytes for 128 logits of them, 8 bytes for 16 with alternatives, and the
    targets' logits; distillation keeps 16 bytes for 128 logits of each row, and 12 bytes and a count for 128 words beside each entry."""
    lib = _lib.load()
    T, V, d = 65536, 131072, 64
    logits = 2 * T * V
    a = _score(T, V, d)
    rows = 8192 * V
    assert lib.swx_logprob_fwd_workspace_bytes(a) <= rows / 8 + 4 * 8192 + 4096
    a.top_k = 20
    assert lib.swx_logprob_fwd_workspace_bytes(a) <= rows / 8 + rows / 2 + 4 * 8192 + 4096
    assert lib.swx_logprob_bwd_workspace_bytes(a) < logits / 16 + 4 * T * d
    b = _distill(T, V, d)
    assert lib.swx_distill_saved_bytes(b) <= T * (12 + 12 * 4 + V / 128 + 17) + 4096
    assert lib.swx_distill_fwd_workspace_bytes(b) < logits / 8 and lib.swx_distill_bwd_workspace_bytes(b) < logits / 16 + 4 * T * d


def test_empty_calls_need_no_buffers():
    lib = _lib.load()
    assert lib.swx_logprob_fwd(_score(T=0), None) == _lib.SWX_OK and lib.swx_token_logprob(_score(T=0), None) == _lib.SWX_OK


def test_cpu_tensors_are_rejected():
    x, w, y = torch.randn(3, 8), torch.randn(5, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        linear_log_probs(x, w, y)
    with pytest.raises(RuntimeError):
        token_log_probs(x)
    with pytest.raises(RuntimeError):
        linear_distillation(x, w, y[:, None], torch.zeros(3, 1))
    with pytest.raises(ValueError):
        linear_distillation(x, w, y[:, None], torch.zeros(3, 1), reduction="max")


def test_a_head_with_a_bias_is_refused():
    model = SiftLM(SiftConfig(vocab_size=20, d_model=8, n_layers=1))
    model.lm_head.bias = torch.nn.Parameter(torch.zeros(20))
    idx = torch.zeros(1, 2, dtype=torch.int64)
    with pytest.raises(ValueError):
        model.log_probs(idx, idx)
    with pytest.raises(ValueError):
        model.distillation_loss(idx, idx[..., None], torch.zeros(1, 2, 1))


def test_distillation_takes_8192_rows_at_a_time():
    """16 bytes for 128 logits of those rows, a sum for four rows of all, whatever the number of tokens."""
    lib = _lib.load()
    V = 131072
    for T in (8192, 65536, 1 << 20):
        assert lib.swx_distill_fwd_workspace_bytes(_distill(T, V, 64)) <= 8192 * V / 8 + 4 * T + 4096


@pytest.mark.parametrize("k,error", [(21, ValueError), (-1, ValueError), (1 << 40, ValueError), (3, RuntimeError)])
def test_generation_refuses_before_it_consumes_the_prompt(k, error, monkeypatch):
    model = SiftLM(SiftConfig(vocab_size=20, d_model=8, n_layers=1))
    steps = []
    monkeypatch.setattr(SiftLM, "step", lambda *a: steps.append(a) or torch.zeros(1, 20))
    for new in (0, 2):
        with pytest.raises(error):
            model.generate(torch.zeros(1, 5, dtype=torch.int64), new, log_probs=k)
    assert not steps
    assert model.generate(torch.zeros(1, 5, dtype=torch.int64), 2).shape == (1, 7)


def test_few_rows_backward_has_room_for_its_statistics():
    """Up to 8 bf16 rows of a large vocabulary: statistics of 128 logits each, which the forward's other products do not give."""
    lib = _lib.load()
    a = _score(T=8, V=5001, d=64)
    b = _distill(T=8, V=5001, d=64)                                              # the same products without them
    assert lib.swx_logprob_bwd_workspace_bytes(a) - lib.swx_distill_bwd_workspace_bytes(b) >= 8 * 2 * 20 * 16 + 5 * 8 * 4
    assert lib.swx_logprob_bwd_workspace_bytes(_score(T=9, V=5001, d=64)) == lib.swx_distill_bwd_workspace_bytes(_distill(T=9, V=5001, d=64))
    a.targets = a.row_max = a.row_sum = a.dx = a.workspace = 4096
    a.workspace_bytes = lib.swx_logprob_bwd_workspace_bytes(a) - 1
    assert lib.swx_logprob_bwd(a, None) == INVALID
