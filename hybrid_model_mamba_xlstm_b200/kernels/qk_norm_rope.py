"""RMS norms of the heads of q and k with the position rotation, over the hxm C ABI.

Does the per-head norms of mLSTMBlock.forward (hybrid_xmamba/layers/
mlstm_block.py:113-114) for q and k at once and turns pairs of the result by
position-dependent angles in the same HBM pass.
"""
from __future__ import annotations

import ctypes
import math

import torch

from .. import _lib
from ._common import dtype_code, no_tangents, on_device, once_only, require_cuda, stream_of

__all__ = ["qk_norm_rope", "qk_norm_rope_bwd"]

_fwd_args, _bwd_args = _lib.packer(_lib.QkNormRopeArgs), _lib.packer(_lib.QkNormRopeBwdArgs)
_FWD, _BWD = ctypes.sizeof(_lib.QkNormRopeArgs), ctypes.sizeof(_lib.QkNormRopeBwdArgs)


_IO = (torch.bfloat16, torch.float32, torch.float16)


def _unit(t):
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _f32(w):
    """A weight as the kernels read it.  A 16-bit one is widened at every call, on the call's stream: a copy kept
    between calls would be blind to writes through .data and to those of other streams and replayed graphs."""
    return w if w is None or (w.dtype == torch.float32 and w.is_contiguous()) else w.detach().float().contiguous()


def _fill(who, q, k, qw, kw, positions, base, rotary, interleaved, eps):
    """(args of the forward with new dense outputs, these, tensors to keep alive)."""
    if q.dim() != 4 or k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
        raise ValueError(f"{who}: q must be (B, L, Hq, d) and k (B, L, Hk, d), got {tuple(q.shape)}, {tuple(k.shape)}")
    if q.dtype not in _IO or k.dtype != q.dtype:
        raise TypeError(f"{who}: q and k must both be fp32, bf16 or fp16, got {q.dtype}, {k.dtype}")
    bsz, L, hq, d = q.shape
    hk = k.shape[2]
    if qw is not None and qw.shape != (d,):
        raise ValueError(f"{who}: q_weight must be ({d},), got {tuple(qw.shape)}")
    if kw is not None and kw.shape != (d,):
        raise ValueError(f"{who}: k_weight must be ({d},), got {tuple(kw.shape)}")
    rotary = (d - d % 2 if positions is not None else 0) if rotary is None else int(rotary)
    if rotary < 0 or rotary > d or rotary % 2:
        raise ValueError(f"{who}: rotary_dim must be even and at most {d}, got {rotary}")
    if not 0 <= eps < math.inf:
        raise ValueError(f"{who}: eps must be finite and at least 0, got {eps}")
    qw, kw = _f32(qw), _f32(kw)
    at = (0, 0, 0)
    if rotary:
        if positions is None:
            raise ValueError(f"{who}: a rotation needs positions")
        if not 0 < base < math.inf:
            raise ValueError(f"{who}: rope_base must be positive and finite, got {base}")
        if positions.dtype != torch.int64:
            if positions.is_floating_point() or positions.dtype == torch.bool:
                raise ValueError(f"{who}: positions must be integers, got {positions.dtype}")
            positions = positions.long()
        if positions.shape == (bsz, L):
            at = (positions.data_ptr(), *positions.stride())
        elif positions.shape == (L,):
            at = (positions.data_ptr(), 0, positions.stride(0))
        else:
            raise ValueError(f"{who}: positions must be ({bsz}, {L}) or ({L},), got {tuple(positions.shape)}")
    q, k = _unit(q), _unit(k)
    yq = torch.empty_like(q, memory_format=torch.contiguous_format)
    yk = torch.empty_like(k, memory_format=torch.contiguous_format)
    a = _fwd_args(_FWD, bsz, L, hq, hk, d, rotary, dtype_code(q), bool(interleaved),
                  q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3],
                  0 if qw is None else qw.data_ptr(), 0 if kw is None else kw.data_ptr(), *at, base, eps,
                  yq.data_ptr(), L * hq * d, hq * d, d, yk.data_ptr(), L * hk * d, hk * d, d)
    return a, yq, yk, (q, k, qw, kw, positions)


def _forward(q, k, qw, kw, positions, base, rotary, interleaved, eps):
    who = "qk_norm_rope"
    dev = require_cuda(q, k, qw, kw, positions, who=who)
    with on_device(dev):
        a, yq, yk, keep = _fill(who, q, k, qw, kw, positions, base, rotary, interleaved, eps)
        _lib.call("hxm_qk_norm_rope_fwd", a, stream_of(dev))
    return yq, yk


def qk_norm_rope_bwd(q, k, q_weight, k_weight, dq_out, dk_out, positions=None, *, rope_base=10000.0, rotary_dim=None,
                     interleaved=False, eps=1e-6, weight_grads=True):
    """Gradients of :func:`qk_norm_rope` for the gradients of its two results.  Returns (dq, dk, dq_weight,
    dk_weight): the first two in q's dtype, the weights' fp32 (None for a weight that is None, or without
    ``weight_grads``)."""
    who = "qk_norm_rope_bwd"
    no_tangents(who, q, k, q_weight, k_weight, dq_out, dk_out)
    dev = require_cuda(q, k, q_weight, k_weight, dq_out, dk_out, positions, who=who)
    if dq_out.shape != q.shape or dk_out.shape != k.shape or dq_out.dtype != q.dtype or dk_out.dtype != k.dtype:
        raise ValueError(f"{who}: the gradients must match q and k")
    with on_device(dev):
        f, dq, dk, keep = _fill(who, q, k, q_weight, k_weight, positions, rope_base, rotary_dim, interleaved, eps)
        dq_out, dk_out = _unit(dq_out), _unit(dk_out)
        dw = [torch.empty_like(w) if weight_grads and w is not None else None for w in keep[2:4]]
        a = _bwd_args(bytes(f), _BWD, dq_out.data_ptr(), *dq_out.stride()[:3], dk_out.data_ptr(), *dk_out.stride()[:3],
                      0 if dw[0] is None else dw[0].data_ptr(), 0 if dw[1] is None else dw[1].data_ptr(), 0, 0)
        n = _lib.lib().hxm_qk_norm_rope_bwd_workspace_size(a)
        ws = torch.empty(n, device=dev, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), n
        _lib.call("hxm_qk_norm_rope_bwd", a, stream_of(dev))
    return dq, dk, dw[0], dw[1]


class QkNormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, positions, base, rotary, interleaved, eps):
        ctx.save_for_backward(q, k, qw, kw, positions)
        ctx.rest = (base, rotary, interleaved, eps)
        return _forward(q, k, qw, kw, positions, base, rotary, interleaved, eps)

    @staticmethod
    def backward(ctx, dyq, dyk):
        once_only("qk_norm_rope")
        q, k, qw, kw, positions = ctx.saved_tensors
        base, rotary, interleaved, eps = ctx.rest
        weights = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        dq, dk, dqw, dkw = qk_norm_rope_bwd(q, k, qw, kw, dyq, dyk, positions, rope_base=base, rotary_dim=rotary,
                                            interleaved=interleaved, eps=eps, weight_grads=weights)
        cast = lambda g, w: None if g is None else g.to(w.dtype)
        return dq, dk, cast(dqw, qw), cast(dkw, kw), None, None, None, None, None


def qk_norm_rope(q, k, q_weight=None, k_weight=None, positions=None, *, rope_base=10000.0, rotary_dim=None,
                 interleaved=False, eps=1e-6):
    """RMS norm over the last dim of every head of q (B, L, Hq, d) and k (B, L, Hk, d), then the rotation of
    its first ``rotary_dim`` elements (default: all with positions, none without) by the position of the
    token: pair p turns by positions * rope_base**(-2p / rotary_dim), where a pair is elements p and
    p + rotary_dim/2, or 2p and 2p + 1 with ``interleaved``.  Differentiable (once) in q, k and the weights.

    q, k: fp32, bf16 or fp16, read in place with any strides that have a unit last one (the column blocks of
    one projection's output); weights (d,) or None (ones); positions (B, L) or (L,) integers, the angles
    formed in 64 bits.  d <= 1024; eps at least 0 (0: a row of zeros gives NaN, as the formula does).  Returns
    the two results, dense, in q's dtype."""
    no_tangents("qk_norm_rope", q, k, q_weight, k_weight)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        return QkNormRopeFunction.apply(q, k, q_weight, k_weight, positions, rope_base, rotary_dim, interleaved, eps)
    return _forward(q, k, q_weight, k_weight, positions, rope_base, rotary_dim, interleaved, eps)
