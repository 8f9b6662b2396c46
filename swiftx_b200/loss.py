"""Losses of the language model's head without its logits: softmax cross entropy, and distillation
from a teacher's top logits.

The reference's training forward multiplies the final norm's output with the head's weight
and hands the fp32 logits to ``F.cross_entropy`` (models/sift_model.py:103-113): two
(tokens, vocab) tensors, and a third for their gradient.  ``linear_cross_entropy`` computes
the same loss and gradients from the two operands; it keeps two floats per token, and one
piece of the vocabulary's logit gradients while the backward runs.  ``linear_distillation`` does so for
the divergence from a teacher's softmax over a few words for each token (no reference counterpart).
"""
import torch
from torch.autograd import forward_ad

from . import _lib

_DT = {torch.float32: 0, torch.bfloat16: 1}


def _rows(t):
    """(n, d) with unit element stride and non-overlapping rows (a copy otherwise)."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def check_operands(name, x, weight, weight16, *others):
    """Checks of a head's operands; returns x as the kernels take it (cast under bf16 autocast)."""
    if not all(t.is_cuda for t in (x, weight, *others)):
        raise RuntimeError(f"swiftx_b200 {name} runs on CUDA tensors only (no CPU path)")
    if any(t.device != x.device for t in (weight, *others)):
        raise ValueError(f"{name}: tensors on {', '.join(str(t.device) for t in (x, weight, *others))}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"{name}: x (..., d) and weight (vocab, d) expected, got {tuple(x.shape)} "
                         f"and {tuple(weight.shape)}")
    if x.dtype == torch.float32 and torch.is_autocast_enabled("cuda") \
            and torch.get_autocast_dtype("cuda") == torch.bfloat16:
        x = x.to(torch.bfloat16)
    if x.dtype not in _DT or weight.dtype not in _DT or (x.dtype == torch.float32 and weight.dtype != torch.float32):
        raise ValueError(f"{name}: fp32 x and weight, or bf16 x with a bf16 or fp32 weight expected, got "
                         f"{x.dtype} and {weight.dtype}")
    if weight16 is not None and (weight16.dtype != torch.bfloat16 or weight16.shape != weight.shape or weight16.device != x.device):
        raise ValueError(f"{name}: weight16 is a bf16 copy of the {tuple(weight.shape)} weight, got {weight16.dtype} "
                         f"{tuple(weight16.shape)}")
    return x


def check_head(name, x, weight, targets, weight16):
    """check_operands, and int64 targets of one for each row of x."""
    x = check_operands(name, x, weight, weight16, targets)
    if targets.dtype != torch.int64 or targets.shape != x.shape[:-1]:
        raise ValueError(f"{name}: int64 targets of shape {tuple(x.shape[:-1])} expected, got "
                         f"{targets.dtype} {tuple(targets.shape)}")
    return x


def check_temperature(name, temperature):
    if not 1e-15 <= temperature <= 1e15:
        raise ValueError(f"{name}: a temperature above 0 (1e-15 to 1e15) expected, got {temperature}")


def product_weight(x, weight, weight16):
    """The weight in x's type."""
    return weight if weight.dtype == x.dtype else weight.to(x.dtype) if weight16 is None else weight16


def set_operands(a, x, w):
    """tokens, vocab, dim, dtype and the operands of an argument struct."""
    a.tokens, a.dim, a.vocab, a.dtype = x.shape[0], x.shape[1], w.shape[0], _DT[x.dtype]
    # a single row's stride may be anything
    a.x, a.x_sr = x.data_ptr(), x.stride(0) if a.tokens != 1 else a.dim
    a.weight, a.w_sr = w.data_ptr(), w.stride(0) if a.vocab != 1 else a.dim


def _args(x, w, targets, ignore_index, reduction):
    a = _lib.XentArgs()
    set_operands(a, x, w)
    a.reduction, a.ignore_index = reduction, ignore_index
    a.targets = targets.data_ptr()
    return a


def _bytes(lib, name, a):
    n = getattr(lib, name)(a)
    if n < 0:
        _lib.check(-n, name)
    return n


def _workspace(lib, name, a, like):
    n = _bytes(lib, name, a)
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
        x, w, targets = _rows(x), _rows(product_weight(x, weight, weight16)), targets.contiguous()
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
    x = check_head("linear_cross_entropy", x, weight, targets, weight16)
    # (a reshape that changes nothing would still be a node of the autograd graph)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    t1 = targets if targets.dim() == 1 else targets.reshape(-1)
    opts = (int(ignore_index), _lib.XENT_REDUCTIONS[reduction])
    if _lib.needs_node(x, weight):
        loss = LinearCrossEntropyFn.apply(x2, weight, t1, *opts, weight16)
    else:
        loss = _forward(_rows(x2), _rows(product_weight(x2, weight, weight16)), t1.contiguous(), *opts)[0]
    return loss.view(targets.shape) if reduction == "none" and targets.dim() != 1 else loss


def _distill_args(x, w, entries, temperature, reduction):
    a = _lib.DistillArgs()
    set_operands(a, x, w)
    a.entries, a.reduction, a.temperature = entries, reduction, temperature
    return a


def _distill_forward(x, w, ids, logits, temperature, reduction):
    """The loss, what the backward needs of it, and the count."""
    T = int(x.shape[0])                # (under a trace a size is a tensor)
    with _lib.on_device(x.device):
        lib = _lib.load()
        loss = x.new_empty((T,) if reduction == _lib.XENT_REDUCTIONS["none"] else (), dtype=torch.float32)
        count = torch.empty_like(loss) if loss.dim() == 0 else loss
        a = _distill_args(x, w, ids.shape[1], temperature, reduction)
        a.teacher_dtype = _DT[logits.dtype]
        a.teacher_ids, a.ids_sr = ids.data_ptr(), ids.stride(0)
        a.teacher_logits, a.tl_sr = logits.data_ptr(), logits.stride(0)
        a.loss, a.count = loss.data_ptr(), count.data_ptr()
        a.saved_bytes = _bytes(lib, "swx_distill_saved_bytes", a)
        saved = x.new_empty(a.saved_bytes, dtype=torch.uint8)
        a.saved = saved.data_ptr()
        ws = _workspace(lib, "swx_distill_fwd_workspace_bytes", a, loss)  # noqa: F841
        _lib.check(lib.swx_distill_fwd(a, _lib.stream_ptr(x.device)), "swx_distill_fwd")
    return loss, saved, count


class LinearDistillationFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, ids, logits, temperature, reduction, weight16=None):
        x, w = _rows(x), _rows(product_weight(x, weight, weight16))
        loss, saved, count = _distill_forward(x, w, ids, logits, temperature, reduction)
        ctx.save_for_backward(x, w, saved, count if count is not loss else None)
        ctx.opts = (ids.shape[1], temperature, reduction, weight.dtype)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, w, saved, count = ctx.saved_tensors
        *opts, w_dtype = ctx.opts
        dloss = dloss.float().contiguous()
        with _lib.on_device(x.device):
            lib = _lib.load()
            dx = torch.empty_like(x, memory_format=torch.contiguous_format) if ctx.needs_input_grad[0] else None
            dw = w.new_empty(w.shape, dtype=w_dtype) if ctx.needs_input_grad[1] else None
            a = _distill_args(x, w, *opts)
            a.saved, a.saved_bytes = saved.data_ptr(), saved.numel()
            a.count = count.data_ptr() if count is not None else None
            a.dw_dtype, a.dloss = _DT[w_dtype], dloss.data_ptr()
            a.dx = dx.data_ptr() if dx is not None else None
            a.dweight = dw.data_ptr() if dw is not None else None
            ws = _workspace(lib, "swx_distill_bwd_workspace_bytes", a, dloss)  # noqa: F841
            _lib.check(lib.swx_distill_bwd(a, _lib.stream_ptr(x.device)), "swx_distill_bwd")
        return dx, dw, None, None, None, None, None


def linear_distillation(x, weight, teacher_ids, teacher_logits, temperature=1.0, reduction="mean", weight16=None):
    """Divergence of a head's softmax from a teacher's over its top words, without the student's logits (CUDA only).

    x (..., d) and weight (vocab, d) as for ``linear_cross_entropy``; teacher_ids (..., K) int64 and
    teacher_logits (..., K) fp32 or bf16, K up to 128: a teacher's largest logits, or log probabilities (a shift of a row
    changes nothing), as ``linear_log_probs(..., top_k=K)`` returns them.  With q a row's softmax of
    teacher_logits / temperature over its used entries and p the student's softmax of logits / temperature over the
    vocabulary, a row's loss is temperature^2 sum_j q_j (log q_j - log p[teacher_ids_j]) (the factor keeps the gradients'
    size).  An entry with an id below 0 or a logit of -inf is not used; a row without used entries does not count.
    Returns the fp32 loss: its mean over the rows that count, their sum, or (reduction "none") one
    value for each row, 0 where nothing counts.

    The types of the gradients, weight16, autocast, dual numbers and traces: as for ``linear_cross_entropy``; the student's logits and
    their accuracy: as for ``linear_log_probs``.  An id of vocab or more, or a teacher logit of NaN or +inf, in a used entry gives a NaN loss
    (and gradients).  The teacher is a constant: a teacher_logits that requires gradients is refused.
    Deterministic."""
    if reduction not in _lib.XENT_REDUCTIONS:
        raise ValueError(f"linear_distillation: reduction {reduction!r}: one of none, mean, sum expected")
    x = check_operands("linear_distillation", x, weight, weight16, teacher_ids, teacher_logits)
    K = teacher_ids.shape[-1] if teacher_ids.dim() else 0
    if teacher_ids.dtype != torch.int64 or teacher_logits.dtype not in _DT or teacher_ids.shape != teacher_logits.shape \
            or teacher_ids.shape[:-1] != x.shape[:-1] or teacher_ids.dim() != x.dim():
        raise ValueError(f"linear_distillation: int64 teacher_ids and fp32 or bf16 teacher_logits of shape {tuple(x.shape[:-1])} + (K,) "
                         f"expected, got {teacher_ids.dtype} {tuple(teacher_ids.shape)} and {teacher_logits.dtype} {tuple(teacher_logits.shape)}")
    if not 1 <= K <= _lib.SWX_MAX_TOP:
        raise ValueError(f"linear_distillation: 1 to {_lib.SWX_MAX_TOP} entries for each row expected, got {K}")
    check_temperature("linear_distillation", temperature)
    if (torch.is_grad_enabled() and teacher_logits.requires_grad) or forward_ad.unpack_dual(teacher_logits).tangent is not None:
        raise RuntimeError("linear_distillation is not differentiable in teacher_logits: detach it")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    ids, logits = (t if t.dim() == 2 else t.reshape(-1, K) for t in (teacher_ids, teacher_logits))
    ids, logits = (t if t.stride(1) == 1 else t.contiguous() for t in (ids, logits))
    opts = (float(temperature), _lib.XENT_REDUCTIONS[reduction])
    if _lib.needs_node(x, weight):
        loss = LinearDistillationFn.apply(x2, weight, ids, logits, *opts, weight16)
    else:
        loss = _distill_forward(_rows(x2), _rows(product_weight(x2, weight, weight16)), ids, logits, *opts)[0]
    return loss.view(x.shape[:-1]) if reduction == "none" and x.dim() != 2 else loss
