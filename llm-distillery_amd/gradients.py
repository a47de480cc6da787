"""The norm of the gradients of all parameters together, and the gradients clipped by it.  Thin wrappers over the C ABI; all arithmetic runs in
the HIP kernels."""
from __future__ import annotations

from array import array
from operator import attrgetter
from typing import Iterable, Optional

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .ops import _DT, _dev, _on, _stream_ptr


_DTYPE = attrgetter("dtype")


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill their stretch of memory, in any order and each place once."""
    want = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


class _Tensors:
    """Tensors as the C ABI takes them: host arrays of addresses, sizes and dtypes."""

    def __init__(self, grads: Iterable[torch.Tensor]):
        self.all = grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
        if not grads:
            raise RuntimeError("no gradients")
        try:
            self.dev = dev = grads[0].device
            usual = {*map(torch.Tensor.get_device, grads)} == {dev.index} and all(map(torch.Tensor.is_contiguous, grads))
        except (AttributeError, TypeError):
            raise RuntimeError("gradients must be tensors (leave out parameters that have none)") from None
        for g in grads if not usual else ():
            if g.device != dev or not g.is_cuda or g.layout is not torch.strided:
                _dev(g, "a gradient", dev if dev.type == "cuda" else None)
                raise RuntimeError("gradients must be dense tensors")
            if not g.is_contiguous() and g.numel() and not _dense(g):
                raise RuntimeError("a gradient must fill its memory (a slice or an expanded tensor does not)")
        try:
            kinds = [*{*map(_DTYPE, grads)}]                   # (most often one)
            self.dtypes = array("i", [_DT[kinds[0]]]) * len(grads) if len(kinds) == 1 else array("i", [_DT[g.dtype] for g in grads])
        except KeyError:
            raise RuntimeError("gradients must be bf16/fp16/fp32") from None
        self.at = array("q", [*map(torch.Tensor.data_ptr, grads)])
        self.sizes = array("q", [*map(torch.Tensor.numel, grads)])

    def args(self):
        return self.at.buffer_info()[0], self.sizes.buffer_info()[0], self.dtypes.buffer_info()[0], len(self.at)

    def workspace(self, lib) -> torch.Tensor:
        return torch.empty(lib.dl_grad_norm_workspace_bytes(self.sizes.buffer_info()[0], len(self.at)), dtype=torch.uint8, device=self.dev)


def _positive(scale: float) -> float:
    scale = float(scale)
    if not 0.0 < scale <= 3.0e38:
        raise ValueError("scale must be positive and finite")
    return scale


def grad_norm(grads: Iterable[torch.Tensor], *, scale: float = 1.0) -> torch.Tensor:
    """`scale` times the 2-norm of all elements of `grads` (bf16/fp16/fp32 tensors of any shapes on one device) together, an fp32 tensor without
    dimensions.  Squares are added up in fp64, in an order that does not change between calls."""
    scale = _positive(scale)
    t = _Tensors(grads)
    lib = _lib.load()
    norm = torch.empty((), dtype=torch.float32, device=t.dev)
    ws = t.workspace(lib)
    with _on(t.dev):
        st = lib.dl_grad_norm(*t.args(), scale, norm.data_ptr(), ws.data_ptr(), ws.numel(), _stream_ptr(t.dev))
    _lib.check(st, "dl_grad_norm")
    return norm


def clip_grads(grads: Iterable[torch.Tensor], max_norm: float, *, scale: float = 1.0, norm: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Multiplies all `grads` in place with `scale` (an average that should be a sum, a loss scale taken out) and, where the norm of what that gives is
    above `max_norm`, with max_norm / norm as well: one factor, one rounding.  Returns the norm before clipping, an fp32 tensor without dimensions.

    `norm` (fp32, one element, `scale` included): is taken for the norm instead, for gradients of which these are only a part (shards on other
    cards: the root of the sum of the squares of their `grad_norm`).  A norm that is NaN or infinite leaves all gradients as they are; one within
    max_norm leaves them unwritten where scale is 1.  The gradients must not overlap.  Autograd takes all of them for written: a backward pass that needs
    what was there raises.  Nothing waits for the GPU."""
    scale, max_norm = _positive(scale), float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must not be negative")
    t = _Tensors(grads)
    lib = _lib.load()
    given = norm is not None
    if given:
        if norm.device != t.dev or norm.dtype != torch.float32 or norm.numel() != 1:
            _dev(norm, "norm")
            raise RuntimeError(f"norm must be one fp32 element on {t.dev}")
        ws = None
    else:
        norm = torch.empty((), dtype=torch.float32, device=t.dev)
        ws = t.workspace(lib)
    with _on(t.dev):
        st = lib.dl_clip_grads(*t.args(), scale, max_norm, norm.data_ptr(), int(given), ws.data_ptr() if ws is not None else 0,
                               ws.numel() if ws is not None else 0, _stream_ptr(t.dev))
    _lib.check(st, "dl_clip_grads")
    increment_version(t.all)
    return norm
