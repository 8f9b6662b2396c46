"""Softmax cross entropy of the language model's head without its logits.

The reference's training forward multiplies the final norm's output with the head's weight
and hands the fp32 logits to ``F.cross_entropy`` (models/sift_model.py:103-113): two
(tokens, vocab) tensors, and a third for their gradient.  ``linear_cross_entropy`` computes
the same loss and gradients from the two operands; it keeps two floats per token, and one
piece of the vocabulary's logit gradients while the backward runs.
"""
import torch

from . import _lib

_DT = {torch.float32: 0, torch.bfloat16: 1}


def _rows(t):
    """(n, d) with unit element stride and non-overlapping rows (a copy otherwise)."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _args(x, w, targets, ignore_index, reduction):
    a = _lib.XentArgs()
    a.tokens, a.dim, a.vocab = x.shape[0], x.shape[1], w.shape[0]
    a.dtype, a.reduction, a.ignore_index = _DT[x.dtype], reduction, ignore_index
    # a single row's stride may be anything
    a.x, a.x_sr = x.data_ptr(), x.stride(0) if a.tokens != 1 else a.dim
    a.weight, a.w_sr = w.data_ptr(), w.stride(0) if a.vocab != 1 else a.dim
    a.targets = targets.data_ptr()
    return a


def _workspace(lib, name, a, like):
    n = getattr(lib, name)(a)
    if n < 0:
        _lib.check(-n, name)
    ws = like.new_empty(n // 4 + 1)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
    return ws


def _forward(x, w, targets, ignore_index, reduction):
    """(loss, (row maxima, reciprocal row sums, count) in one buffer) of checked operands."""
    T = int(x.shape[0])                # (under a trace a size is a tensor)
    with _lib.on_device(x.device):
        lib = _lib.load()
        none = reduction == _lib.XENT_REDUCTIONS["none"]
        loss = x.new_empty((T,) if none else (), dtype=torch.float32)
        stats = loss.new_empty(2 * T + 1)
        a = _args(x, w, targets, ignore_index, reduction)
        a.loss = loss.data_ptr()
        a.row_max = stats.data_ptr()
        a.row_rsum, a.count = a.row_max + 4 * T, a.row_max + 8 * T
        ws = _workspace(lib, "swx_xent_fwd_workspace_bytes", a, loss)  # noqa: F841
        _lib.check(lib.swx_xent_fwd(a, _lib.stream_ptr(x.device)), "swx_xent_fwd")
    return loss, stats


class LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, ignore_index, reduction, weight16=None):
        w = weight if weight.dtype == x.dtype else weight.to(x.dtype) if weight16 is None else weight16
        x, w, targets = _rows(x), _rows(w), targets.contiguous()
        loss, stats = _forward(x, w, targets, ignore_index, reduction)
        ctx.save_for_backward(x, w, targets, stats)
        ctx.opts = (ignore_index, reduction, weight.dtype)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, w, targets, stats = ctx.saved_tensors
        ignore_index, reduction, w_dtype = ctx.opts
        dloss = dloss.float().contiguous()
        with _lib.on_device(x.device):
            lib = _lib.load()
            dx = torch.empty_like(x, memory_format=torch.contiguous_format) if ctx.needs_input_grad[0] else None
            dw = w.new_empty(w.shape, dtype=w_dtype) if ctx.needs_input_grad[1] else None
            a = _args(x, w, targets, ignore_index, reduction)
            a.row_max = stats.data_ptr()
            a.row_rsum, a.count = a.row_max + 4 * x.shape[0], a.row_max + 8 * x.shape[0]
            a.dw_dtype, a.dloss = _DT[w_dtype], dloss.data_ptr()
            a.dx = dx.data_ptr() if dx is not None else None
            a.dweight = dw.data_ptr() if dw is not None else None
            ws = _workspace(lib, "swx_xent_bwd_workspace_bytes", a, stats)  # noqa: F841
            _lib.check(lib.swx_xent_bwd(a, _lib.stream_ptr(x.device)), "swx_xent_bwd")
        return dx, dw, None, None, None, None


def linear_cross_entropy(x, weight, targets, ignore_index=-100, reduction="mean", weight16=None):
    """``F.cross_entropy(F.linear(x, weight).float(), targets)`` without the logits (CUDA only).

    x (..., d) and weight (vocab, d), fp32 or bf16; targets (...) int64.  Returns the fp32
    loss: its mean over the tokens that count, their sum, or (reduction "none") one value
    for each token, 0 at ignored ones.  bf16 operands give the products of bf16 values summed in
    fp32 in the tensor cores (losses 2e-7 off at a width of 1024; the error grows with the width, as a library product's does),
    and the logits' gradient is rounded to bf16 once for its products with the weight and x (gradients 2.0e-3 off in the
    mean square at a vocabulary of 256, where their own rounding alone gives 1.7e-3; no difference at 50001).  fp32
    operands keep fp32 accuracy and have to be finite (an infinity gives NaN).  With bf16 x an fp32 weight is rounded
    to bf16 for the products (what autocast's linear does) and its gradient comes back in fp32, not
    rounded; under bf16 autocast an fp32 x is cast too.  The gradients are deterministic.

    A target outside [0, vocab) other than ignore_index gives a NaN loss (and gradients)
    instead of a device-side assertion; x has to be finite in ignored rows too.  Forward-mode dual numbers are
    refused, and torch.jit.trace records the call as a Python operator.  weight16: a bf16
    copy of an fp32 weight that the caller keeps (used with bf16 x instead of rounding again)."""
    if reduction not in _lib.XENT_REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction {reduction!r}: one of none, mean, sum expected")
    if not (x.is_cuda and weight.is_cuda and targets.is_cuda):
        raise RuntimeError("swiftx_b200 linear_cross_entropy runs on CUDA tensors only (no CPU path)")
    if x.device != weight.device or x.device != targets.device:
        raise ValueError(f"linear_cross_entropy: tensors on {x.device}, {weight.device} and {targets.device}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"linear_cross_entropy: x (..., d) and weight (vocab, d) expected, got {tuple(x.shape)} "
                         f"and {tuple(weight.shape)}")
    if targets.dtype != torch.int64 or targets.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: int64 targets of shape {tuple(x.shape[:-1])} expected, got "
                         f"{targets.dtype} {tuple(targets.shape)}")
    if x.dtype == torch.float32 and torch.is_autocast_enabled("cuda") \
            and torch.get_autocast_dtype("cuda") == torch.bfloat16:
        x = x.to(torch.bfloat16)
    if x.dtype not in _DT or weight.dtype not in _DT or (x.dtype == torch.float32 and weight.dtype != torch.float32):
        raise ValueError(f"linear_cross_entropy: fp32 x and weight, or bf16 x with a bf16 or fp32 weight expected, got "
                         f"{x.dtype} and {weight.dtype}")
    if weight16 is not None and (weight16.dtype != torch.bfloat16 or weight16.shape != weight.shape or weight16.device != x.device):
        raise ValueError(f"linear_cross_entropy: weight16 is a bf16 copy of the {tuple(weight.shape)} weight, got {weight16.dtype} "
                         f"{tuple(weight16.shape)}")
    # (a reshape that changes nothing would still be a node of the autograd graph)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    t1 = targets if targets.dim() == 1 else targets.reshape(-1)
    opts = (int(ignore_index), _lib.XENT_REDUCTIONS[reduction])
    if _lib.needs_node(x, weight):
        loss = LinearCrossEntropyFn.apply(x2, weight, t1, *opts, weight16)
    else:
        w = weight if weight.dtype == x.dtype else weight.to(x.dtype) if weight16 is None else weight16
        loss = _forward(_rows(x2), _rows(w), t1.contiguous(), *opts)[0]
    return loss.view(targets.shape) if reduction == "none" and targets.dim() != 1 else loss
