"""What a student needs to write its own continuations: sampling from its logits, and its head in 8-bit floating point.  Thin
wrappers over the C ABI; all arithmetic runs in the HIP kernels."""
from __future__ import annotations

from typing import NamedTuple, Tuple, Union

import torch

from . import _lib
from .ops import _DT, _dev, _on, _row_pitch, _rows_2d, _stream_ptr


def _setting(value, n: int, dtype: torch.dtype, name: str, dev: torch.device):
    """(pointer, value for all rows, what keeps the memory alive) of a setting: a number, or a vector with one entry per row."""
    if not isinstance(value, torch.Tensor):
        return 0, value, None
    _dev(value, name, dev)
    if value.dtype != dtype or value.numel() != n:
        raise RuntimeError(f"{name} must be a number or a {dtype} tensor with one entry for each of the {n} rows")
    v = value.reshape(-1).contiguous()
    return v.data_ptr(), 0, v


def sample_rows(logits: torch.Tensor, u: torch.Tensor, *, temperature: Union[float, torch.Tensor] = 1.0,
                top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
                min_p: Union[float, torch.Tensor] = 0.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """One token for every row of logits [..., V] (bf16/fp16/fp32, rows evenly strided) from a random number in [0, 1) per row,
    `u` fp32.

    The tokens of a row are taken in descending order of their logits (equal logits: the lower index first) with the weights
    softmax(logits / temperature).  `top_k` > 0 keeps the first k; `top_p` < 1 of those the shortest beginning that has at least
    top_p of their mass; `min_p` > 0 what comes ahead of the first token with less than min_p times the largest probability.  The
    token is the one in whose stretch of the kept mass u falls.  A temperature of 0 (or below) takes the first maximum.  Each
    setting is a number, or a tensor with one entry per row (fp32; top_k int32).

    Weights are whole numbers, 2^31 for the most likely token, so the choice is exact: the same logits and the same u give the same
    token however the rows are batched.  u counts with 24 bits.  NaN and -inf logits are never drawn.

    Returns (tokens int64, logp fp32, kept int32) of shape logits.shape[:-1]: the token, its log-probability under
    softmax(logits / temperature) before any filter, and how many tokens the filters kept.  A row without a finite logit (nor
    +inf) gives (-1, -inf, 0)."""
    _dev(logits, "logits")
    if logits.dim() == 1:
        return tuple(t[0] for t in sample_rows(logits.unsqueeze(0), u.reshape(1), temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p))
    x = _rows_2d(logits)
    R, V = x.shape
    dev = x.device
    if x.dtype not in _DT:
        raise RuntimeError("unsupported dtype")
    _dev(u, "u", dev)
    if u.dtype != torch.float32 or u.numel() != R:
        raise RuntimeError(f"u must be an fp32 tensor with one entry for each of the {R} rows")
    u = u.reshape(-1).contiguous()
    if V == 0:
        raise RuntimeError("the rows have no columns")
    T, T0, keep_T = _setting(temperature, R, torch.float32, "temperature", dev)
    k, k0, keep_k = _setting(top_k, R, torch.int32, "top_k", dev)
    p, p0, keep_p = _setting(top_p, R, torch.float32, "top_p", dev)
    m, m0, keep_m = _setting(min_p, R, torch.float32, "min_p", dev)
    k0 = int(k0)
    if not 0 <= k0 <= 0x7fffffff:
        raise ValueError("top_k must not be negative")
    tokens = torch.empty(R, dtype=torch.int64, device=dev)
    logp = torch.empty(R, dtype=torch.float32, device=dev)
    kept = torch.empty(R, dtype=torch.int32, device=dev)
    with _on(dev):
        st = _lib.load().dl_sample_rows(x.data_ptr(), _DT[x.dtype], _row_pitch(x), R, V, u.data_ptr(), T, k, p, m, float(T0), k0, float(p0),
                                        float(m0), tokens.data_ptr(), logp.data_ptr(), kept.data_ptr(), _stream_ptr(dev))
    _lib.check(st, "dl_sample_rows")
    shape = logits.shape[:-1]
    return tokens.view(shape), logp.view(shape), kept.view(shape)
