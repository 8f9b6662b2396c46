"""Log probabilities of given tokens, with the entropy and the top alternatives.

The reference makes logits (models/sift_model.py:107, 115) and leaves what is read out of them to its
callers.  ``linear_log_probs`` computes a token's log probability, the entropy and the largest alternatives from the head's two
operands, with gradients and without (tokens, vocab) logits; ``token_log_probs`` from the logits of a step of generation.
"""
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .loss import _DT, _rows, _workspace, check_head, check_temperature, product_weight, set_operands


class LogProbs(NamedTuple):
    """What scoring returns: fp32 log_probs and entropy of the tokens' shape, and with top_k the fp32
    top_log_probs and int64 top_ids with a last dimension of top_k (None otherwise)."""
    log_probs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_log_probs: Optional[torch.Tensor] = None
    top_ids: Optional[torch.Tensor] = None


def _outputs(a, like, T, top_k, with_log_probs=True):
    """(log_probs, entropy, top_log_probs, top_ids), set in the argument struct."""
    ent = like.new_empty(T, dtype=torch.float32)
    a.entropy = ent.data_ptr()
    lp = vals = ids = None
    if with_log_probs:
        lp = torch.empty_like(ent)
        a.log_probs = lp.data_ptr()
    if top_k:
        vals, ids = ent.new_empty((T, top_k)), ent.new_empty((T, top_k), dtype=torch.int64)
        a.top_log_probs, a.top_ids = vals.data_ptr(), ids.data_ptr()
    return lp, ent, vals, ids


def _args(x, w, targets, ignore_index, top_k, temperature):
    a = _lib.LogprobArgs()
    set_operands(a, x, w)
    a.top_k, a.temperature, a.ignore_index, a.targets = top_k, temperature, ignore_index, targets.data_ptr()
    return a


def _forward(x, w, targets, opts, keep):
    """The outputs and, when asked for, the rows' maxima and sums in one buffer."""
    T = int(x.shape[0])                # (under a trace a size is a tensor)
    with _lib.on_device(x.device):
        lib = _lib.load()
        a = _args(x, w, targets, *opts)
        out = _outputs(a, x, T, opts[1])
        stats = out[1].new_empty(2 * T + 1) if keep else None      # (never empty: it has an address)
        if keep:
            a.row_max = stats.data_ptr()
            a.row_sum = a.row_max + 4 * T
        ws = _workspace(lib, "swx_logprob_fwd_workspace_bytes", a, out[1])  # noqa: F841
        _lib.check(lib.swx_logprob_fwd(a, _lib.stream_ptr(x.device)), "swx_logprob_fwd")
    return out, stats


class LinearLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, ignore_index, top_k, temperature, weight16=None):
        x, w, targets = _rows(x), _rows(product_weight(x, weight, weight16)), targets.contiguous()
        opts = (ignore_index, top_k, temperature)
        out, stats = _forward(x, w, targets, opts, True)
        ctx.save_for_backward(x, w, targets, stats, out[1])
        ctx.opts = (opts, weight.dtype)
        ctx.set_materialize_grads(False)
        if not top_k:
            return out[:2]
        ctx.mark_non_differentiable(*out[2:])
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlp, dent, *_):
        x, w, targets, stats, entropy = ctx.saved_tensors
        opts, w_dtype = ctx.opts
        if dlp is None and dent is None:
            return (None,) * 7
        dlp, dent = (t.float().contiguous() if t is not None else None for t in (dlp, dent))
        with _lib.on_device(x.device):
            lib = _lib.load()
            dx = torch.empty_like(x, memory_format=torch.contiguous_format) if ctx.needs_input_grad[0] else None
            dw = w.new_empty(w.shape, dtype=w_dtype) if ctx.needs_input_grad[1] else None
            a = _args(x, w, targets, *opts)
            a.row_max, a.entropy = stats.data_ptr(), entropy.data_ptr()
            a.row_sum, a.dw_dtype = a.row_max + 4 * x.shape[0], _DT[w_dtype]
            a.d_log_probs, a.d_entropy, a.dx, a.dweight = (t.data_ptr() if t is not None else None for t in (dlp, dent, dx, dw))
            ws = _workspace(lib, "swx_logprob_bwd_workspace_bytes", a, stats)  # noqa: F841
            _lib.check(lib.swx_logprob_bwd(a, _lib.stream_ptr(x.device)), "swx_logprob_bwd")
        return dx, dw, None, None, None, None, None


def check_top(name, top_k, vocab):
    if not 0 <= top_k <= min(vocab, _lib.SWX_MAX_TOP):
        raise ValueError(f"{name}: top_k of 0 to {min(vocab, _lib.SWX_MAX_TOP)} expected, got {top_k}")


def linear_log_probs(x, weight, targets, top_k=0, temperature=1.0, ignore_index=-100, weight16=None):
    """Log probabilities of ``targets`` under softmax(F.linear(x, weight) / temperature), the entropy of that
    softmax, and its top_k largest alternatives, without the logits (CUDA only).  Returns ``LogProbs``.

    x (..., d), weight (vocab, d), targets (...) int64, weight16 and autocast as for ``linear_cross_entropy``; top_k up to
    128.  log_probs (at most 0) and entropy are differentiable in x and weight (a gradient of one alone may be asked for);
    the alternatives are not.  Ignored tokens: zeros, ids of -1 and no gradient, whatever x holds there as long as it is
    finite.  Alternatives are in falling order, the lowest word first among equals; they are ordered by products of the
    operands good to 2^-45 of their magnitudes (fp32 operands: summed in fp64), so that rounding changes neither
    their order nor their ties (among the top_k + 4 or more words with the largest fp32 products: where more words than that
    differ by a rounding of those, others of them may be missing).

    bf16 operands: products summed in fp32 in the tensor cores (8192 terms at a time), the logits' gradient rounded to bf16
    once for its products.  The tensor cores' additions cut off; the exponents' scale makes up for the mean of that,
    0.23 2^-24 of the logits for each 16 terms, which the loss does not do (a sum that loses nothing, as a one-hot row's, comes out too
    large by as much, 9e-7 at a width of 1024).  fp32 operands keep fp32 accuracy and have to be finite.  A target outside
    [0, vocab) other than ignore_index gives NaN, and so does a row with a NaN or +inf logit, or with nothing but -inf.  Dual
    numbers are refused, torch.jit.trace records a Python operator.  Deterministic."""
    x = check_head("linear_log_probs", x, weight, targets, weight16)
    check_top("linear_log_probs", top_k, weight.shape[0])
    check_temperature("linear_log_probs", temperature)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    t1 = targets if targets.dim() == 1 else targets.reshape(-1)
    opts = (int(ignore_index), int(top_k), float(temperature))
    if _lib.needs_node(x, weight):
        out = LinearLogProbsFn.apply(x2, weight, t1, *opts, weight16)
    else:
        out, _ = _forward(_rows(x2), _rows(product_weight(x2, weight, weight16)), t1.contiguous(), opts, False)
    if targets.dim() != 1:
        out = tuple(t if t is None else t.view(targets.shape + t.shape[1:]) for t in out)
    return LogProbs(*out)


def token_log_probs(logits, targets=None, top_k=0, temperature=1.0, ignore_index=-100):
    """``linear_log_probs`` from logits (..., vocab), fp32 or bf16, such as ``SiftLM.step`` returns (CUDA only).
    Without targets log_probs is None.

    Logits of -inf are words that are not allowed (probability 0).  A row with a NaN or +inf, or with nothing but -inf, gives
    NaN values and ids in order all the same (NaNs first).  Not differentiable: logits that require gradients are
    refused unless gradients are disabled, dual numbers and torch.jit.trace always."""
    if not logits.is_cuda or (targets is not None and not targets.is_cuda):
        raise RuntimeError("swiftx_b200 token_log_probs runs on CUDA tensors only (no CPU path)")
    if logits.dtype not in _DT or logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"token_log_probs: fp32 or bf16 logits (..., vocab) expected, got {logits.dtype} {tuple(logits.shape)}")
    if targets is not None and (targets.dtype != torch.int64 or targets.shape != logits.shape[:-1] or targets.device != logits.device):
        raise ValueError(f"token_log_probs: int64 targets of shape {tuple(logits.shape[:-1])} on {logits.device} expected, got "
                         f"{targets.dtype} {tuple(targets.shape)} on {targets.device}")
    check_top("token_log_probs", top_k, logits.shape[-1])
    check_temperature("token_log_probs", temperature)
    if _lib.needs_node(logits):
        if torch.jit.is_tracing():
            raise RuntimeError("token_log_probs cannot be traced: its launch would not be recorded")
        if (torch.is_grad_enabled() and logits.requires_grad) or forward_ad.unpack_dual(logits).tangent is not None:
            raise RuntimeError("token_log_probs is not differentiable: call it under no_grad, or linear_log_probs on the head's operands")
    z = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    z = z if z.stride(1) == 1 or z.shape[1] == 1 else z.contiguous()
    with _lib.on_device(z.device):
        lib = _lib.load()
        a = _lib.LogprobArgs()
        a.tokens, a.vocab, a.dtype, a.x, a.x_sr = z.shape[0], z.shape[1], _DT[z.dtype], z.data_ptr(), z.stride(0)
        a.top_k, a.temperature, a.ignore_index = top_k, temperature, ignore_index
        t1 = None
        if targets is not None:
            t1 = (targets if targets.dim() == 1 else targets.reshape(-1)).contiguous()
            a.targets = t1.data_ptr()
        out = _outputs(a, z, z.shape[0], top_k, targets is not None)
        _lib.check(lib.swx_token_logprob(a, _lib.stream_ptr(z.device)), "swx_token_logprob")
    if logits.dim() != 2:
        out = tuple(t if t is None else t.view(logits.shape[:-1] + t.shape[1:]) for t in out)
    return LogProbs(*out)
