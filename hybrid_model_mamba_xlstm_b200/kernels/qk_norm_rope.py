"""RMS norms of the heads of q and k with the position rotation, over the hxm C ABI.

Does the per-head norms of mLSTMBlock.forward (hybrid_xmamba/layers/
mlstm_block.py:113-114) for q and k at once and turns pairs of the result by
position-dependent angles in the same HBM pass.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from ._common import dtype_code, f32_param, on_device, once_only, ptr, require_cuda, stream_of

__all__ = ["qk_norm_rope", "qk_norm_rope_bwd"]

_fwd_args, _bwd_args = _lib.packer(_lib.QkNormRopeArgs), _lib.packer(_lib.QkNormRopeBwdArgs)
_FWD, _BWD = ctypes.sizeof(_lib.QkNormRopeArgs), ctypes.sizeof(_lib.QkNormRopeBwdArgs)


def _unit(t):
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _fill(who, q, k, qw, kw, positions, base, rotary, interleaved, eps):
    """(args of the forward with new dense outputs, these, tensors to keep alive)."""
    if q.dim() != 4 or k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"{who}: q must be (B, L, Hq, d) and k (B, L, Hk, d), got {tuple(q.shape)}, {tuple(k.shape)}")
    if q.dtype not in (torch.float32, torch.bfloat16, torch.float16) or k.dtype != q.dtype:
        raise TypeError(f"{who}: q and k must both be fp32, bf16 or fp16, got {q.dtype}, {k.dtype}")
    bsz, L, hq, d = q.shape
    for name, w in (("q_weight", qw), ("k_weight", kw)):
        if w is not None and w.shape != (d,):
            raise ValueError(f"{who}: {name} must be ({d},), got {tuple(w.shape)}")
    rotary = (d - d % 2 if positions is not None else 0) if rotary is None else int(rotary)
    if rotary < 0 or rotary > d or rotary % 2:
        raise ValueError(f"{who}: rotary_dim must be even and at most {d}, got {rotary}")
    if rotary and positions is None:
        raise ValueError(f"{who}: a rotation needs positions")
    if rotary and not (base > 0 and base < float("inf")):
        raise ValueError(f"{who}: rope_base must be positive and finite, got {base}")
    q, k = _unit(q), _unit(k)
    qw, kw = f32_param(qw), f32_param(kw)
    at = (0, 0, 0)
    if rotary:
        if positions.is_floating_point() or positions.dtype == torch.bool or positions.shape not in ((bsz, L), (L,)):
            raise ValueError(f"{who}: positions must be integers ({bsz}, {L}) or ({L},), got {positions.dtype} "
                             f"{tuple(positions.shape)}")
        positions = positions.long()
        at = (positions.data_ptr(), *(positions.stride() if positions.dim() == 2 else (0, positions.stride(0))))
    yq = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    yk = torch.empty(k.shape, device=q.device, dtype=q.dtype)
    a = _fwd_args(_FWD, bsz, L, hq, k.shape[2], d, rotary, dtype_code(q), bool(interleaved),
                  q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3], ptr(qw) or 0, ptr(kw) or 0, *at,
                  float(base), float(eps), yq.data_ptr(), *yq.stride()[:3], yk.data_ptr(), *yk.stride()[:3])
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
    dev = require_cuda(q, k, q_weight, k_weight, dq_out, dk_out, positions, who=who)
    if dq_out.shape != q.shape or dk_out.shape != k.shape or dq_out.dtype != q.dtype or dk_out.dtype != k.dtype:
        raise ValueError(f"{who}: the gradients must match q and k")
    with on_device(dev):
        f, dq, dk, keep = _fill(who, q, k, q_weight, k_weight, positions, rope_base, rotary_dim, interleaved, eps)
        dq_out, dk_out = _unit(dq_out), _unit(dk_out)
        d = q.shape[-1]
        dw = [torch.empty(d, device=dev, dtype=torch.float32) if weight_grads and w is not None else None
              for w in (q_weight, k_weight)]
        a = _bwd_args(bytes(f), _BWD, dq_out.data_ptr(), *dq_out.stride()[:3], dk_out.data_ptr(), *dk_out.stride()[:3],
                      ptr(dw[0]) or 0, ptr(dw[1]) or 0, 0, 0)
        n = _lib.lib().hxm_qk_norm_rope_bwd_workspace_size(a)
        ws = torch.empty(n, device=dev, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ptr(ws), n
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
    formed in 64 bits.  d <= 1024.  Returns the two results, dense, in q's dtype."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return QkNormRopeFunction.apply(q, k, q_weight, k_weight, positions, rope_base, rotary_dim, interleaved, eps)
    return _forward(q, k, q_weight, k_weight, positions, rope_base, rotary_dim, interleaved, eps)
