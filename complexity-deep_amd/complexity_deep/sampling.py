"""Choosing the next token on the gfx950 kernel (models/modeling.py:258-283).

``sample_tokens`` is the temperature, top-k and top-p sampling of ``generate`` with min-p beside
them, from random numbers that the caller gives: one launch, no sort, nothing read back.  Weights are
summed as 64-bit integers (cdx_sample_tokens), so that a token never depends on the order in
which threads add; equal logits count in the order of their indices.
"""

from __future__ import annotations

import math
from typing import Union

import torch

from . import _native as nat

Setting = Union[float, torch.Tensor]

MAX_VOCAB = 1 << 20


def _setting(v: Setting, B: int, like: torch.Tensor, name: str, top: float, dtype: torch.dtype):
    """(pointer or None, scalar, tensor kept alive) of one setting."""
    if isinstance(v, torch.Tensor):
        if v.dtype != dtype or tuple(v.shape) != (B,) or v.device != like.device:
            raise ValueError(f"sample_tokens: {name} must be a number or a {dtype} tensor of shape ({B},) on "
                             f"{like.device}, got {v.dtype} {tuple(v.shape)} on {v.device}")
        v = v if v.is_contiguous() else v.contiguous()
        return v.data_ptr(), 0, v
    if not 0 <= v <= top or not math.isfinite(v):
        raise ValueError(f"sample_tokens: {name}={v} is out of range")
    if dtype == torch.int32:
        if int(v) != v:
            raise ValueError(f"sample_tokens: {name}={v} must be an integer")
        return None, min(int(v), MAX_VOCAB), None
    return None, float(v), None


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature: Setting = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Setting = 1.0, min_p: Setting = 0.0) -> torch.Tensor:
    """One token (int64 [B]) per row of ``logits`` [B, V] (bf16 or fp32), drawn with ``uniforms`` [B]
    (fp32 in [0, 1)).

    With w_i = exp((x_i - max x) / temperature): top_k keeps the logits that reach the k-th largest;
    top_p keeps, in descending order and by index among equals, the tokens before which the sum is
    at most top_p of the total; min_p keeps w_i >= min_p.  The token is the first index whose running sum
    of kept weights exceeds uniforms * their total.

    Each setting is a number or a tensor with one value per row (int32 for top_k, fp32 for the
    others).  temperature 0 takes the first maximum; top_k 0, top_p 1 and min_p 0 cut nothing.  In
    a tensor, a temperature or top_k below 0 counts as 0, top_p outside [0, 1] as the nearer end,
    min_p above 1 as 1.  A NaN logit counts as -inf; a row of -inf alone gives -1."""
    fast = nat.host()
    if fast is not None:
        tokens = fast.sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p)
        if tokens is not None:
            return tokens
    what = "sample_tokens"
    nat.require_device(logits, uniforms, dtype=None, what=what)
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{what}: logits must be bf16 or fp32 [rows, vocab], got {logits.dtype} {tuple(logits.shape)}")
    B, V = logits.shape
    if not 0 < V <= MAX_VOCAB:
        raise ValueError(f"{what}: a vocabulary of {V} (1 .. {MAX_VOCAB} supported)")
    if uniforms.dtype != torch.float32 or tuple(uniforms.shape) != (B,):
        raise ValueError(f"{what}: uniforms must be fp32 [{B}], got {uniforms.dtype} {tuple(uniforms.shape)}")
    t = _setting(temperature, B, logits, "temperature", 3e38, torch.float32)
    k = _setting(top_k, B, logits, "top_k", math.inf, torch.int32)
    p = _setting(top_p, B, logits, "top_p", 1.0, torch.float32)
    m = _setting(min_p, B, logits, "min_p", 1.0, torch.float32)
    ld = logits.stride(0) if B > 1 else V
    if (V > 1 and logits.stride(1) != 1) or ld < V:
        logits, ld = logits.contiguous(), V
    uniforms = uniforms if uniforms.is_contiguous() else uniforms.contiguous()
    tokens = torch.empty(B, dtype=torch.int64, device=logits.device)
    with nat.on_device(logits), nat.launch_region("sample", logits.device, B=B, V=V):
        nat.check(nat.lib().cdx_sample_tokens(
            logits.data_ptr(), logits.dtype == torch.float32, ld, B, V, uniforms.data_ptr(), t[0], t[1], k[0], k[1],
            p[0], p[1], m[0], m[1], tokens.data_ptr(), nat.stream_of(logits)), "cdx_sample_tokens")
    return tokens
