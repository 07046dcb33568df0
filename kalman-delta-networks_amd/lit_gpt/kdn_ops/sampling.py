"""Sampling one token per row of logits from given random numbers (``kdn_sample``).

The reference has no counterpart: it evaluates whole sequences and generates nothing.
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import _lib

MAX_VOCAB = 1 << 20
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _finite(v):
    return 0 <= v < math.inf


def _count(v):
    return isinstance(v, int) and v >= 0


def _share(v):
    return 0 < v <= 1


def _part(v):
    return 0 <= v <= 1


# The kernel's scalars are fp32: a number past its range is taken as its nearest positive one (a temperature or top_p of
# 1e-50 is not 0).
_TINY, _MAX = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max


def _positive(v) -> float:
    return float(v) if _TINY <= v <= _MAX or v == 0 else _TINY if v < 1 else _MAX


def _setting(name: str, value, rows: int, dtype, ok, what: str):
    """(tensor or None, scalar) of a per-call or per-row setting."""
    if isinstance(value, torch.Tensor):
        if value.shape != (rows,) or value.dtype != dtype:
            raise ValueError(f"{name} must be a number or {dtype} [{rows}], got {value.dtype} {tuple(value.shape)}")
        return (value if value.is_contiguous() else value.contiguous()), 0
    if not ok(value):
        raise ValueError(f"{name} must be {what}, got {value!r}")
    return None, value


def sample_tokens(logits: torch.Tensor, noise: Optional[torch.Tensor], *, temperature: Union[float, torch.Tensor] = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
                  min_p: Union[float, torch.Tensor] = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """``(tokens [rows] int64, logprobs [rows] fp32)`` for ``logits`` [rows, vocab] (bf16, fp16 or fp32).

    ``noise`` [rows, vocab] fp32 holds the random numbers, positive and from Exp(1) (``torch.empty(...).exponential_()``).
    With p = softmax(logits / temperature) and the tokens in the order (logit descending, index ascending), these are
    kept: the first ``top_k`` (0: all); of them the shortest prefix that holds ``top_p`` of their mass (1: all); of them
    those with p >= ``min_p`` times the largest.  The token is argmax p / noise over the kept, which is distributed as p
    restricted to them; its log-probability is that of p, before any truncation.

    Each setting is a number, or a tensor [rows] (fp32; ``top_k`` int32) with one for each row.  ``temperature`` 0 takes
    the largest logit (lowest index), with the log-probability at temperature 1; if it is 0 for the whole call ``noise``
    may be None.  Tokens whose logit is -inf or NaN are never drawn; a row with no other gets token -1, logprob -inf.

    There is no derivative: inputs that require a gradient (while autograd is on) or carry a tangent are refused."""
    if logits.ndim != 2:
        raise ValueError(f"logits must be [rows, vocab], got {tuple(logits.shape)}")
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"logits must be bf16, fp16 or fp32, got {logits.dtype}")
    B, V = logits.shape
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"the vocabulary must have 1 to {MAX_VOCAB} tokens, got {V}")
    t_rows, t = _setting("temperature", temperature, B, torch.float32, _finite, "finite and >= 0")
    k_rows, k = _setting("top_k", top_k, B, torch.int32, _count, "an integer >= 0")
    p_rows, p = _setting("top_p", top_p, B, torch.float32, _share, "in (0, 1]")
    m_rows, m = _setting("min_p", min_p, B, torch.float32, _part, "in [0, 1]")
    if noise is None:
        if t_rows is not None or t != 0:
            raise ValueError("noise is needed unless temperature is 0")
    elif noise.shape != (B, V) or noise.dtype != torch.float32:
        raise ValueError(f"noise must be fp32 [{B}, {V}], got {noise.dtype} {tuple(noise.shape)}")
    _lib.refuse_derivatives("sample_tokens", logits, noise, t_rows, p_rows, m_rows)
    _lib.one_device(logits, noise, t_rows, k_rows, p_rows, m_rows)
    dev = logits.device
    if (V > 1 and logits.stride(1) != 1) or (B > 1 and logits.stride(0) < V):
        logits = logits.contiguous()
    if noise is not None and ((V > 1 and noise.stride(1) != 1) or (B > 1 and noise.stride(0) < V)):
        noise = noise.contiguous()
    tokens = torch.empty((B,), device=dev, dtype=torch.int64)
    logprobs = torch.empty((B,), device=dev, dtype=torch.float32)
    if B:
        with _lib.on(dev):
            _lib.call("kdn_sample", logits.data_ptr(), code, logits.stride(0), _lib.ptr(noise),
                      0 if noise is None else noise.stride(0), _lib.ptr(t_rows), _positive(t), _lib.ptr(k_rows), min(k, V),
                      _lib.ptr(p_rows), _positive(p), _lib.ptr(m_rows), float(m), B, V, tokens.data_ptr(),
                      logprobs.data_ptr(), _lib.stream_of(logits))
    return tokens, logprobs


__all__ = ("sample_tokens",)
