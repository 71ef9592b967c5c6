"""Token sampling over the hxm C ABI: the sampling rule of HybridLanguageModel.generate
(hybrid_xmamba/models/hybrid_lm.py:238-262) in one launch, from given uniform numbers."""
from __future__ import annotations

import ctypes
import math

import torch

from .. import _lib
from ._common import dtype_code, on_device, require_cuda, stream_of

__all__ = ["sample_tokens"]

_args, _SIZE = _lib.packer(_lib.SampleArgs), ctypes.sizeof(_lib.SampleArgs)


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
    rows = [x for x in (temperature, top_k, top_p, min_p) if isinstance(x, torch.Tensor)]
    dev = require_cuda(logits, uniforms, *rows, who=who)
    if logits.dim() != 2 or uniforms.shape != logits.shape[:1]:
        raise ValueError(f"{who}: logits must be (B, V) and uniforms (B,), got {tuple(logits.shape)}, {tuple(uniforms.shape)}")
    bsz, vocab = logits.shape
    if vocab < 1:
        raise ValueError(f"{who}: empty vocabulary")
    with on_device(dev):
        keep = []  # the settings' tensors as the kernel reads them

        def setting(name, x, off, most):
            """(number, address of the numbers of the rows or 0)"""
            if isinstance(x, torch.Tensor):
                if x.shape != (bsz,):
                    raise ValueError(f"{who}: {name} must be a number or ({bsz},), got {tuple(x.shape)}")
                if name == "top_k":
                    if x.is_floating_point() or x.dtype == torch.bool:
                        raise TypeError(f"{who}: top_k must be integers, got {x.dtype}")
                    x = x if x.dtype == torch.int32 else x.long().clamp(0, vocab).int()  # the type may not hold vocab
                keep.append((x if name == "top_k" else x.float()).contiguous())
                return off, keep[-1].data_ptr()
            if x is None:
                return off, 0
            if name == "top_k":
                if x != int(x) or x < 0:
                    raise ValueError(f"{who}: top_k must be a whole number of at least 0, got {x}")
                return min(int(x), vocab), 0
            if not 0 <= x <= most:
                raise ValueError(f"{who}: {name} must be at least 0{'' if name == 'temperature' else ' and at most 1'}, got {x}")
            return ctypes.c_float(x).value, 0

        settings = (*setting("temperature", temperature, 1.0, math.inf), *setting("top_k", top_k, 0, None),
                    *setting("top_p", top_p, 1.0, 1), *setting("min_p", min_p, 0.0, 1))
        if vocab > 1 and logits.stride(1) != 1:
            logits = logits.contiguous()
        if uniforms.dtype != torch.float32 or not uniforms.is_contiguous():
            uniforms = uniforms.float().contiguous()
        tokens = torch.empty_like(uniforms, dtype=torch.int64)
        logprob = torch.empty_like(uniforms) if return_logprob else None
        a = _args(_SIZE, bsz, vocab, dtype_code(logits), logits.data_ptr(), logits.stride(0), uniforms.data_ptr(), *settings,
                  tokens.data_ptr(), logprob.data_ptr() if return_logprob else 0)
        _lib.call("hxm_sample_tokens", a, stream_of(dev))
    return (tokens, logprob) if return_logprob else tokens
