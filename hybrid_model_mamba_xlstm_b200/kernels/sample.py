"""Token sampling over the hxm C ABI: the sampling rule of HybridLanguageModel.generate
(hybrid_xmamba/models/hybrid_lm.py:238-262) in one launch, from given uniform numbers."""
from __future__ import annotations

import torch

from .. import _lib
from ._common import dtype_code, on_device, ptr, require_cuda, stream_of

__all__ = ["sample_tokens"]


def sample_tokens(logits, uniforms, *, temperature=1.0, top_k=None, top_p=None, min_p=None, return_logprob=False):
    """One token (int64) for each row of ``logits`` (B, V) from its number of ``uniforms`` (B,), fp32 in [0, 1).

    With x = logits / temperature and weights w = exp(x - max x) in 64 bits: ``top_k`` keeps the k largest
    logits (None or 0: all), ``top_p`` of these the ones that, by falling logit, have at most top_p of the
    weight before them (the first always; None or 1: all), ``min_p`` of these the ones with w >= min_p.
    Equal logits rank by rising token.  The token is the first kept one, in rising order, up to which the
    weights exceed uniforms * their total.  temperature 0 takes the largest logit (the lowest token of equal
    ones).  Logits of -inf and NaN are never taken, +inf ones share all of the weight, and a row without any
    other logit gives -1.  Each setting is a number, or a (B,) tensor with one per row (there: temperature
    not above 0 is greedy, top_k below 1 keeps all); settings count as fp32.

    logits: fp32, bf16 or fp16 with a unit last stride (others are copied), V <= 2^18.  Returns tokens (B,)
    [and the log-probability of each under the kept tokens, fp32: 0 when greedy, -inf for -1]."""
    who = "sample_tokens"
    rows = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    tensors = {n: x for n, x in rows.items() if isinstance(x, torch.Tensor)}
    dev = require_cuda(logits, uniforms, *tensors.values(), who=who)
    if logits.dim() != 2 or uniforms.shape != logits.shape[:1]:
        raise ValueError(f"{who}: logits must be (B, V) and uniforms (B,), got {tuple(logits.shape)}, {tuple(uniforms.shape)}")
    bsz, vocab = logits.shape
    if vocab < 1:
        raise ValueError(f"{who}: empty vocabulary")
    a = _lib.SampleArgs()
    a.rows, a.vocab, a.io_dtype = bsz, vocab, dtype_code(logits)
    off = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    with on_device(dev):
        keep = []
        for n, x in rows.items():
            if n in tensors:
                if x.shape != (bsz,):
                    raise ValueError(f"{who}: {n} must be a number or ({bsz},), got {tuple(x.shape)}")
                if n == "top_k" and (x.is_floating_point() or x.dtype == torch.bool):
                    raise TypeError(f"{who}: top_k must be integers, got {x.dtype}")
                x = (x if x.dtype == torch.int32 else x.clamp(0, vocab).int()) if n == "top_k" else x.float()
                x = x.contiguous()
                keep.append(x)
                setattr(a, n + "_rows", x.data_ptr())
                continue
            x = off[n] if x is None else x
            if n == "top_k":
                if x != int(x) or x < 0:
                    raise ValueError(f"{who}: top_k must be a whole number of at least 0, got {x}")
                x = min(int(x), vocab)
            elif not x >= 0 or (n != "temperature" and x > 1):
                raise ValueError(f"{who}: {n} must be at least 0{'' if n == 'temperature' else ' and at most 1'}, got {x}")
            setattr(a, n, x)
        if vocab > 1 and logits.stride(1) != 1:
            logits = logits.contiguous()
        uniforms = uniforms.float().contiguous()
        tokens = torch.empty(bsz, device=dev, dtype=torch.int64)
        logprob = torch.empty(bsz, device=dev, dtype=torch.float32) if return_logprob else None
        a.logits, a.logits_row_stride, a.uniforms = ptr(logits), logits.stride(0), ptr(uniforms)
        a.tokens, a.logprob = ptr(tokens), ptr(logprob)
        _lib.call("hxm_sample_tokens", a, stream_of(dev))
    return (tokens, logprob) if return_logprob else tokens
