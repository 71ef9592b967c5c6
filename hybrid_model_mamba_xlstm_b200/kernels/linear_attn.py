"""Linear attention with a constant decay per head over the hxm C ABI.

The reference has no such kernel; the recurrence is its mLSTM loop
(hybrid_xmamba/kernels/tfla/tfla_interface.py:113-137) with a constant forget
gate and without input gate and normalizer:
    S_t = exp(log_decay_h) S_(t-1) + k_t v_t^T,   o_t = scale * S_t^T q_t.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from ._common import dtype_code, no_tangents, on_device, once_only, require_cuda, stream_of

__all__ = ["linear_attention", "linear_attention_bwd", "linear_attention_step"]

_fwd_args, _bwd_args, _step_args = (_lib.packer(c) for c in (_lib.LinearAttnArgs, _lib.LinearAttnBwdArgs, _lib.LinearAttnStepArgs))
_FWD, _BWD, _STEP = (ctypes.sizeof(c) for c in (_lib.LinearAttnArgs, _lib.LinearAttnBwdArgs, _lib.LinearAttnStepArgs))
_NONE = (0,) * 5  # an absent state: address and strides


def _check_io(who, q, k, v):
    if q.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{who}: q must be fp32 or bf16, got {q.dtype}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{who}: q, k, v must have one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")


def _check(who, q, k, v):
    if q.dim() != 4:
        raise ValueError(f"{who}: q must be (B, L, H, dk), got {tuple(q.shape)}")
    if k.shape != q.shape or v.shape[:-1] != q.shape[:-1] or v.dim() != 4:
        raise ValueError(f"{who}: k must be {tuple(q.shape)} and v (B, L, H, dv), got {tuple(k.shape)}, {tuple(v.shape)}")
    _check_io(who, q, k, v)


def _scale(who, scale, dk):
    scale = dk ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -126 <= abs(scale) <= 2.0 ** 126:  # the gradients divide by it
        raise ValueError(f"{who}: scale must be nonzero, of 2^-126 to 2^126, got {scale}")
    return scale


def _decay(who, log_decay, heads):
    if log_decay.shape != (heads,):
        raise ValueError(f"{who}: log_decay must be ({heads},), got {tuple(log_decay.shape)}")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{who}: log_decay is a constant; it must not require a gradient")
    return log_decay if log_decay.dtype == torch.float32 and log_decay.is_contiguous() else log_decay.float().contiguous()


def _rows(t):
    """t (.., d) as the kernels read it: unit stride in the last dim, 16-byte aligned rows where a
    copy can bring that about (a zero stride repeats data and stays)."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return t.contiguous()
    e = 16 // t.element_size()
    if t.data_ptr() % 16 == 0 and t.is_contiguous():
        return t
    if t.shape[-1] % e == 0 and (t.data_ptr() % 16 or any(s % e for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)):
        return t.contiguous() if not t.is_contiguous() else t.clone()
    return t


def _at(t):
    """Address and strides of t (B, L, H, d); those of extents of 1 count for nothing and are 0."""
    s, n = t.stride(), t.shape
    return t.data_ptr(), s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0


def _fill(who, q, k, v, log_decay, scale, lengths, s0, out, sT, error_flag, wait_limit_cycles):
    """(args of the forward, tensors to keep alive); out and sT: where the backward has none, None."""
    bsz, L, nh, dk = q.shape
    if lengths is not None:
        if lengths.shape != (bsz,) or lengths.is_floating_point() or lengths.dtype == torch.bool:
            raise ValueError(f"{who}: lengths must be ({bsz},) integers")
        if lengths.dtype != torch.int32:
            lengths = lengths.long().clamp(0, L).int()  # widened first: L may be beyond the type's range
        lengths = lengths.contiguous()
    if error_flag is not None and (error_flag.dtype != torch.int32 or error_flag.numel() < 1):
        raise ValueError(f"{who}: error_flag must be an int32 tensor with an element, got {error_flag.dtype} {tuple(error_flag.shape)}")
    if s0 is not None:
        if s0.shape != (bsz, nh, dk, v.shape[-1]):
            raise ValueError(f"{who}: initial_state must be {(bsz, nh, dk, v.shape[-1])}, got {tuple(s0.shape)}")
        s0 = s0.float()
    q, k, v = _rows(q), _rows(k), _rows(v)
    ld = _decay(who, log_decay, nh)
    a = _fwd_args(_FWD, bsz, L, nh, dk, v.shape[-1], dtype_code(q), *_at(q), *_at(k), *_at(v),
                  *(_NONE[:4] if out is None else _at(out)), ld.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
                  *(_NONE if s0 is None else (s0.data_ptr(), *s0.stride())),
                  *(_NONE if sT is None else (sT.data_ptr(), *sT.stride())),
                  scale, 0, 0, 0 if error_flag is None else error_flag.data_ptr(), int(wait_limit_cycles))
    return a, (q, k, v, ld, lengths, s0)


def _forward(q, k, v, log_decay, scale, lengths, s0, want_state, error_flag=None, wait_limit_cycles=0):
    who = "linear_attention"
    dev = require_cuda(q, k, v, log_decay, lengths, s0, error_flag, who=who)
    with on_device(dev):
        _check(who, q, k, v)
        out = torch.empty_like(v, memory_format=torch.contiguous_format)
        sT = torch.empty(q.shape[0], q.shape[2], q.shape[3], v.shape[3], device=dev, dtype=torch.float32) if want_state else None
        a, keep = _fill(who, q, k, v, log_decay, scale, lengths, s0, out, sT, error_flag, wait_limit_cycles)
        n = _lib.lib().hxm_linear_attn_workspace_size(a)
        if n:
            ws = torch.empty(n, device=dev, dtype=torch.uint8)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n
        _lib.call("hxm_linear_attn_fwd", a, stream_of(dev))
    return out, sT


def linear_attention_bwd(q, k, v, log_decay, dout, *, scale=None, lengths=None, initial_state=None, d_final_state=None,
                         need_d_initial_state=None, error_flag=None, wait_limit_cycles=0):
    """Gradients of :func:`linear_attention` for dout (B, L, H, dv) and d_final_state (B, H, dk, dv) or None.

    Returns (dq, dk, dv, d_initial_state): the first three in q's dtype, the last fp32, or None unless
    ``need_d_initial_state`` (default: with an initial_state).  They are three more runs of the same
    recurrence, dk and dv in reversed time, so dv (the size) may be at most 512 like dk."""
    who = "linear_attention_bwd"
    no_tangents(who, q, k, v, log_decay, dout, initial_state, d_final_state)
    dev = require_cuda(q, k, v, log_decay, dout, lengths, initial_state, d_final_state, error_flag, who=who)
    if dout.shape != v.shape or dout.dtype != q.dtype:
        raise ValueError(f"{who}: dout must be {tuple(v.shape)} {q.dtype}, got {tuple(dout.shape)} {dout.dtype}")
    scale = _scale(who, scale, q.shape[-1])
    if need_d_initial_state is None:
        need_d_initial_state = initial_state is not None
    with on_device(dev):
        _check(who, q, k, v)
        f, keep = _fill(who, q, k, v, log_decay, scale, lengths, initial_state, None, None, error_flag, wait_limit_cycles)
        dout = _rows(dout)
        sshape = (q.shape[0], q.shape[2], q.shape[3], v.shape[3])
        if d_final_state is not None:
            if d_final_state.shape != sshape:
                raise ValueError(f"{who}: d_final_state must be {sshape}, got {tuple(d_final_state.shape)}")
            d_final_state = d_final_state.float()
        dq = torch.empty_like(q, memory_format=torch.contiguous_format)
        dk = torch.empty_like(q, memory_format=torch.contiguous_format)
        dv = torch.empty_like(v, memory_format=torch.contiguous_format)
        ds0 = torch.empty(sshape, device=dev, dtype=torch.float32) if need_d_initial_state else None
        a = _bwd_args(bytes(f), _BWD, *_at(dout),
                      *(_NONE if d_final_state is None else (d_final_state.data_ptr(), *d_final_state.stride())),
                      dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), 0 if ds0 is None else ds0.data_ptr(), 0, 0)
        n = _lib.lib().hxm_linear_attn_bwd_workspace_size(a)
        if n:
            ws = torch.empty(n, device=dev, dtype=torch.uint8)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n
        _lib.call("hxm_linear_attn_bwd", a, stream_of(dev))
    return dq, dk, dv, ds0


class LinearAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, s0, log_decay, scale, lengths, want_state, error_flag, wait_limit_cycles):
        ctx.save_for_backward(q, k, v, s0, log_decay, lengths)
        ctx.rest = (scale, error_flag, wait_limit_cycles)
        out, sT = _forward(q, k, v, log_decay, scale, lengths, s0, want_state, error_flag, wait_limit_cycles)
        ctx.set_materialize_grads(False)
        return out, sT

    @staticmethod
    def backward(ctx, dout, dsT):
        once_only("linear_attention")
        q, k, v, s0, log_decay, lengths = ctx.saved_tensors
        if dout is None and dsT is None:
            return (None,) * 10
        scale, error_flag, wait_limit_cycles = ctx.rest
        if dout is None:
            dout = torch.zeros(v.shape, device=v.device, dtype=v.dtype)
        dq, dk, dv, ds0 = linear_attention_bwd(q, k, v, log_decay, dout.to(q.dtype), scale=scale, lengths=lengths,
                                               initial_state=s0, d_final_state=dsT,
                                               need_d_initial_state=s0 is not None and ctx.needs_input_grad[3],
                                               error_flag=error_flag, wait_limit_cycles=wait_limit_cycles)
        return (dq, dk, dv, ds0 if ds0 is None else ds0.to(s0.dtype)) + (None,) * 6


def linear_attention(q, k, v, log_decay, *, scale=None, lengths=None, initial_state=None, return_final_state=False,
                     error_flag=None, wait_limit_cycles=0):
    """Linear attention over whole sequences, from and to a carried state; differentiable (once).

    q, k (B, L, H, dk), v (B, L, H, dv): bf16 or fp32, any strides (views with a unit last stride and
    16-byte aligned rows are read in place, zero strides too, others copied); log_decay (H,) fp32, at
    most 0 (-inf: each step forgets all before it), a constant without a gradient; scale: default
    dk**-0.5, of 2^-126 to 2^126 in size; lengths (B,) integers: only the first lengths[b] steps of row b
    count (held to [0, L]), later rows of the output are zero and their inputs are never used;
    initial_state (B, H, dk, dv).  Returns o (B, L, H, dv) in q's dtype [and the state after the last counted
    step, fp32 (B, H, dk, dv), to continue with this function or :func:`linear_attention_step`].  An infinity
    or NaN among the inputs makes what the recurrence forms from it infinite or NaN (which of them is not
    defined), and nothing else: no earlier step, other head or row.

    dk <= 512, and dv <= 512 for gradients; B <= 21845, H <= 65535, L <= 2^30. bf16 with dk, dv multiples of 8
    and dk <= 256 (for gradients dv <= 256 too) runs on the tensor cores, where the weights of q k and the copy
    of the state that meets q are rounded to bf16 like the inputs (a bf16 result is then off by up to 2^-8 of
    the sum of absolute values besides its own rounding; states and d_initial_state keep 32 bits); everything
    else on the FP32 pipe. error_flag: a device int32 tensor set to 1 if a bounded device wait of the call or of
    its gradients gave up (the outputs are then not valid); wait_limit_cycles: that bound in SM cycles (0: about
    2 s)."""
    who = "linear_attention"
    if q.dim() != 4:
        raise ValueError(f"{who}: q must be (B, L, H, dk), got {tuple(q.shape)}")
    no_tangents(who, q, k, v, initial_state, log_decay)
    scale = _scale(who, scale, q.shape[-1])
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, initial_state, log_decay)):
        if v.shape[-1] > 512:
            raise ValueError(f"{who}: gradients need dv <= 512, got {v.shape[-1]}")
        _decay(who, log_decay, q.shape[2])
        out, sT = LinearAttentionFunction.apply(q, k, v, initial_state, log_decay, scale, lengths, bool(return_final_state),
                                                error_flag, wait_limit_cycles)
    else:
        out, sT = _forward(q, k, v, log_decay, scale, lengths, initial_state, return_final_state, error_flag,
                           wait_limit_cycles)
    return (out, sT) if return_final_state else out


def linear_attention_step(q, k, v, log_decay, state, *, scale=None, out=None):
    """One step for every row: ``state`` (B, H, dk, dv; fp32, unit last stride) becomes
    exp(log_decay) state + k v^T in place, and o = scale * state^T q (B, H, dv) is returned (in ``out``
    if given, which shares no memory with q, k or the state).  q, k (B, H, dk), v (B, H, dv): bf16 or fp32.
    Without gradients."""
    who = "linear_attention_step"
    no_tangents(who, q, k, v, log_decay, state)
    dev = require_cuda(q, k, v, log_decay, state, out, who=who)
    if q.dim() != 3:
        raise ValueError(f"{who}: q must be (B, H, dk), got {tuple(q.shape)}")
    bsz, nh, dk = q.shape
    dv = v.shape[-1]
    if k.shape != q.shape or v.dim() != 3 or v.shape[:2] != q.shape[:2]:
        raise ValueError(f"{who}: k must be {tuple(q.shape)} and v (B, H, dv), got {tuple(k.shape)}, {tuple(v.shape)}")
    _check_io(who, q, k, v)
    if state.shape != (bsz, nh, dk, dv) or state.dtype != torch.float32:
        raise ValueError(f"{who}: state must be fp32 {(bsz, nh, dk, dv)}, got {state.dtype} {tuple(state.shape)}")
    at = state.stride()
    if (dv > 1 and at[3] != 1) or (bsz > 1 and at[0] == 0) or (nh > 1 and at[1] == 0) or (dk > 1 and at[2] == 0):
        raise ValueError(f"{who}: state is updated in place: it needs a unit last stride and no repeated rows")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad
                                    or state.requires_grad or (out is not None and out.requires_grad)):
        raise ValueError(f"{who}: has no gradient; use linear_attention, or torch.no_grad()")
    scale = _scale(who, scale, dk)
    with on_device(dev):
        if dk > 1 and q.stride(2) != 1:
            q = q.contiguous()
        if dk > 1 and k.stride(2) != 1:
            k = k.contiguous()
        if dv > 1 and v.stride(2) != 1:
            v = v.contiguous()
        ld = _decay(who, log_decay, nh)
        written = (state,) if out is None else (state, out)
        if out is None:
            out = torch.empty_like(v, memory_format=torch.contiguous_format)
        elif out.shape != (bsz, nh, dv) or out.dtype != q.dtype or (dv > 1 and out.stride(-1) != 1) or any(
                s == 0 for s, n in zip(out.stride(), out.shape) if n > 1):
            raise ValueError(f"{who}: out must be {q.dtype} {(bsz, nh, dv)} with a unit last stride and no repeated rows")
        a = _step_args(_STEP, bsz, nh, dk, dv, dtype_code(q), q.data_ptr(), *q.stride()[:2], k.data_ptr(), *k.stride()[:2],
                       v.data_ptr(), *v.stride()[:2], out.data_ptr(), *out.stride()[:2], ld.data_ptr(), state.data_ptr(),
                       *at[:3], scale)
        _lib.call("hxm_linear_attn_step", a, stream_of(dev))
    torch.autograd.graph.increment_version(written)  # gradients that need what was there are refused
    return out
