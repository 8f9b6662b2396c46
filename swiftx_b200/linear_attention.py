"""Linear attention with a decay for each head: a recurrence with a matrix state.

Where the selective scan (models/selective_scan.py:34) keeps ``d_state`` values for each
channel, ``linear_attention`` keeps a (dk, dv) matrix for each head:

    S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T,    out_t = scale * S_t^T q_t

Over a sequence it runs chunked, on the tensor cores, with gradients; ``linear_attention_step``
is its form for one token per row, on a state that it updates in place.
"""
import torch
from torch.autograd import forward_ad

from . import _lib

MAX_DIM = 128                    # largest dk and dv
_DT = {torch.float32: 0, torch.bfloat16: 1}


def _unit(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check(name, q, k, v, log_decay, state, lead):
    """Shapes, types and devices of an operand set; ``lead``: the dimensions before the heads, (b) or (b, L)."""
    dev = q.device
    if dev.type != "cuda" or k.device != dev or v.device != dev or log_decay.device != dev \
            or (state is not None and state.device != dev):
        if all(t is None or t.is_cuda for t in (q, k, v, log_decay, state)):
            raise ValueError(f"{name}: tensors on several devices")
        raise RuntimeError(f"swiftx_b200 {name} runs on CUDA tensors only (no CPU path)")
    qs, vs = q.shape, v.shape
    if len(qs) != lead + 2 or len(vs) != lead + 2 or k.shape != qs or vs[:lead] != qs[:lead]:
        raise ValueError(f"{name}: q, k {'(b, Hk, dk)' if lead == 1 else '(b, L, Hk, dk)'} and v with its b"
                         f"{'' if lead == 1 else ', L'} expected, got {tuple(qs)}, {tuple(k.shape)} and {tuple(vs)}")
    hk, dk = qs[lead:]
    h, dv = vs[lead:]
    if hk < 1 or h < 1 or h % hk:
        raise ValueError(f"{name}: v's {h} heads are not a multiple of q's and k's {hk}")
    if not (1 <= dk <= MAX_DIM and 1 <= dv <= MAX_DIM):
        raise ValueError(f"{name}: dk and dv of 1 to {MAX_DIM} expected, got {dk} and {dv}")
    if q.dtype not in _DT or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{name}: q, k and v of one dtype, fp32 or bf16, expected, got {q.dtype}, {k.dtype} and {v.dtype}")
    gs = log_decay.shape
    if log_decay.dtype != torch.float32 or (gs != vs[:-1] and gs != vs[lead:-1]):
        raise ValueError(f"{name}: fp32 log_decay of shape {(h,)} or {tuple(vs[:-1])} expected, got "
                         f"{log_decay.dtype} {tuple(gs)}")
    if state is not None and (state.dtype != torch.float32 or state.shape != (vs[0], h, dk, dv)):
        raise ValueError(f"{name}: fp32 state of shape {(vs[0], h, dk, dv)} expected, got {state.dtype} {tuple(state.shape)}")


def _args(q, k, v, g, scale):
    a = _lib.LinattnArgs()
    a.batch, a.seqlen, a.heads, a.dv = v.shape
    a.qk_heads, a.dk = q.shape[2:]
    a.dtype, a.scale, a.decay_per_head = _DT[q.dtype], scale, int(g.dim() == 1)
    a.q, (a.q_sb, a.q_sl, a.q_sh) = q.data_ptr(), q.stride()[:3]
    a.k, (a.k_sb, a.k_sl, a.k_sh) = k.data_ptr(), k.stride()[:3]
    a.v, (a.v_sb, a.v_sl, a.v_sh) = v.data_ptr(), v.stride()[:3]
    a.log_decay = g.data_ptr()
    a.g_sb, a.g_sl, a.g_sh = (0, 0, g.stride(0)) if g.dim() == 1 else g.stride()
    return a


def _dense(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(q, k, v, g, s0, lengths, scale, want_state, save):
    """(out, the last state or None, the states at the backward's segments' starts or None: with
    ``save``, where there are several) of checked operands."""
    b, _, h, dv = v.shape
    dk = q.shape[-1]
    with _lib.on_device(v.device):
        lib = _lib.load()
        a = _args(q, k, v, g, scale)
        n = lib.swx_linattn_fwd_workspace_bytes(a)
        if n < 0:
            _lib.check(-n, "swx_linattn_fwd")
        out = _dense(v)
        last = g.new_empty((b, h, dk, dv)) if want_state else None
        seg = None
        if n > 0:
            ws = g.new_empty(n // 4)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n
        if save:
            m = lib.swx_linattn_segments(a)
            if m > 1:
                seg = g.new_empty((b, h, m, dk, dv))
                a.seg_states = seg.data_ptr()
        a.lengths, a.initial_state, a.out, a.final_state = _ptr(lengths), _ptr(s0), out.data_ptr(), _ptr(last)
        _lib.check(lib.swx_linattn_fwd(a, _lib.stream_ptr(v.device)), "swx_linattn_fwd")
    return out, last, seg


class LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_state, lengths, scale, want_state):
        out, last, seg = _forward(q, k, v, log_decay, initial_state, lengths, scale, want_state, True)
        ctx.save_for_backward(q, k, v, log_decay, initial_state, lengths, seg)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlast):
        q, k, v, g, s0, lengths, seg = ctx.saved_tensors
        dout = torch.zeros_like(v) if dout is None else _unit(dout.to(v.dtype))
        dlast = dlast.float().contiguous() if dlast is not None else None
        with _lib.on_device(v.device):
            lib = _lib.load()
            a = _args(q, k, v, g, ctx.scale)
            dq, dk, dv, dg = _dense(q), _dense(k), _dense(v), _dense(g)
            ds0 = _dense(s0) if s0 is not None and ctx.needs_input_grad[4] else None
            ws = g.new_empty(lib.swx_linattn_bwd_workspace_bytes(a) // 4)
            a.lengths, a.initial_state, a.seg_states, a.dfinal_state = _ptr(lengths), _ptr(s0), _ptr(seg), _ptr(dlast)
            a.dout, (a.do_sb, a.do_sl, a.do_sh) = dout.data_ptr(), dout.stride()[:3]
            a.dq, a.dk_out, a.dv_out, a.dlog_decay = dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr()
            a.dinitial_state = _ptr(ds0)
            a.workspace, a.workspace_bytes = ws.data_ptr(), 4 * ws.numel()
            _lib.check(lib.swx_linattn_bwd(a, _lib.stream_ptr(v.device)), "swx_linattn_bwd")
        return dq, dk, dv, dg, ds0, None, None, None


def linear_attention(q, k, v, log_decay, initial_state=None, scale=1.0, lengths=None, return_state=False):
    """out_t = scale * S_t^T q_t with S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T (CUDA only).

    q, k (b, L, Hk, dk) and v (b, L, H, dv), all fp32 or all bf16, dk and dv up to 128, with any strides
    and a unit one along the last dimension (a copy otherwise); H a multiple of Hk: head h reads
    q and k of head h // (H // Hk).  log_decay fp32, (b, L, H), or (H,) for fixed decays; 0 keeps
    the state, -inf resets it.  initial_state fp32 (b, H, dk, dv).  lengths, an int64 (b,) tensor:
    row i has lengths[i] tokens (clamped to 0..L); what lies behind them is not used (it may be NaN), gives
    zeros in out and in the gradients, and leaves the state; up to there q, k and v have to be finite (an
    infinity or NaN at one token can reach the outputs of the chunk's earlier tokens).  Returns out (b, L, H, dv),
    and with return_state the fp32 state after the last token.  Differentiable in q, k, v, log_decay and
    initial_state (dual numbers of forward mode are refused, torch.jit.trace records a Python operator);
    deterministic.

    Carried states and log_decay's gradient have fp32 accuracy.  bf16 inputs: the score tiles, and the state where
    it is read out (its gradient, for v's), are rounded to bf16 once for their products, so that a result carries two
    roundings, a term's and its own (2.35e-3 in the mean square, 1.66e-3 with its own alone).  fp32 inputs: products
    of two tf32 pieces, about 22 bits (5e-7 off where fp32 products are 2e-7).

    Gradients where heads share q and k, or with dv above 64, take two fp32 buffers of (b, L, H ceil(dv / 64), dk)."""
    _check("linear_attention", q, k, v, log_decay, initial_state, 2)
    if lengths is not None:
        if lengths.dtype != torch.int64 or tuple(lengths.shape) != (v.shape[0],) or lengths.device != v.device:
            raise ValueError(f"linear_attention: int64 lengths of shape {(v.shape[0],)} on {v.device} expected, got "
                             f"{lengths.dtype} {tuple(lengths.shape)} on {lengths.device}")
        lengths = lengths.contiguous()
    q, k, v = _unit(q), _unit(k), _unit(v)
    if initial_state is not None:
        initial_state = initial_state.contiguous()
    if _lib.needs_node(q, k, v, log_decay, initial_state):
        out, state = LinearAttentionFn.apply(q, k, v, log_decay, initial_state, lengths, float(scale), return_state)
    else:
        out, state, _ = _forward(q, k, v, log_decay, initial_state, lengths, float(scale), return_state, False)
    return (out, state) if return_state else out


def linear_attention_step(q, k, v, log_decay, state, scale=1.0):
    """One token of ``linear_attention`` for every row: q, k (b, Hk, dk), v (b, H, dv), log_decay
    (b, H) or (H,); ``state``, a dense fp32 (b, H, dk, dv) tensor (as linear_attention returns it), is updated
    in place.  Returns out (b, H, dv) in v's dtype.  Not differentiable: operands that require
    gradients are refused unless they are disabled, dual numbers and torch.jit.trace always."""
    _check("linear_attention_step", q, k, v, log_decay, state, 1)
    if not state.is_contiguous():
        raise ValueError("linear_attention_step: state must be a dense (b, H, dk, dv) tensor")
    if _lib.needs_node(q, k, v, log_decay, state):
        if torch.jit.is_tracing():
            raise RuntimeError("linear_attention_step cannot be traced: its update of the state would not be recorded")
        if (torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, log_decay, state))) \
                or any(forward_ad.unpack_dual(t).tangent is not None for t in (q, k, v, log_decay, state)):
            raise RuntimeError("linear_attention_step is not differentiable: call it under no_grad, or linear_attention on one token")
    q, k, v = _unit(q), _unit(k), _unit(v)
    with _lib.on_device(v.device):
        lib = _lib.load()
        out = _dense(v)
        a = _lib.LinattnArgs()
        a.batch, a.heads, a.dv = v.shape
        a.seqlen, (a.qk_heads, a.dk) = 1, q.shape[1:]
        a.dtype, a.scale = _DT[q.dtype], float(scale)
        a.q, (a.q_sb, a.q_sh) = q.data_ptr(), q.stride()[:2]
        a.k, (a.k_sb, a.k_sh) = k.data_ptr(), k.stride()[:2]
        a.v, (a.v_sb, a.v_sh) = v.data_ptr(), v.stride()[:2]
        a.log_decay = log_decay.data_ptr()
        a.g_sb, a.g_sh = (0, log_decay.stride(0)) if log_decay.dim() == 1 else log_decay.stride()
        a.out, a.final_state = out.data_ptr(), state.data_ptr()
        _lib.check(lib.swx_linattn_step(a, _lib.stream_ptr(v.device)), "swx_linattn_step")
    torch.autograd.graph.increment_version(state)      # a backward that saved this state must not use the new one
    return out
