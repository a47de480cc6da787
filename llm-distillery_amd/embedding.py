"""Embedding lookup with a scale, and its gradient by sorted tokens.  Thin wrappers over the C ABI; all arithmetic runs in the
HIP kernels."""
from __future__ import annotations

from typing import Optional

import torch
from torch.utils._python_dispatch import is_in_torch_dispatch_mode

from . import _lib
from .ops import _DT, _IT, _dev, _on, _row_pitch, _share_memory, _stream_ptr


def _tokens_1d(tokens: torch.Tensor, dev: torch.device) -> torch.Tensor:
    _dev(tokens, "tokens", dev)
    if tokens.dtype not in _IT:
        raise RuntimeError("tokens must be int32 or int64")
    return tokens if tokens.dim() == 1 and tokens.is_contiguous() else tokens.reshape(-1).contiguous()


def _matrix(t: torch.Tensor, name: str) -> None:
    if t.dim() != 2 or t.dtype not in _DT:
        raise RuntimeError(f"{name} must be a bf16/fp16/fp32 matrix")
    rows, width = t.shape
    pitch, one = t.stride()
    if rows > 1 and pitch < width or width > 1 and one != 1:
        raise RuntimeError(f"{name} must be dense along its rows")


def embed_rows(table: torch.Tensor, tokens: torch.Tensor, *, scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`scale * table[tokens]` as [*tokens.shape, width], rounded once to the table's dtype.

    table [vocab, width] bf16/fp16/fp32, rows dense, any row stride; tokens int32/int64 of any shape.  A token outside
    [0, vocab) is padding and gives a row of zeros.  `out` [number of tokens, width]: the result is written there."""
    _dev(table, "table")
    _matrix(table, "table")
    dev = table.device
    t = _tokens_1d(tokens, dev)
    n, (V, W) = t.numel(), table.shape
    if out is None:
        res = torch.empty((n, W), dtype=table.dtype, device=dev)
    else:
        res = out
        _dev(out, "out", dev)
        _matrix(out, "out")
        if tuple(out.shape) != (n, W) or out.dtype != table.dtype:
            raise RuntimeError(f"out must be a [{n}, {W}] {table.dtype} matrix")
        if _share_memory(out, table):
            raise RuntimeError("out must not share memory with the table")
    with _on(dev):
        st = _lib.load().dl_embed_rows(table.data_ptr(), _DT[table.dtype], _row_pitch(table), V, W, t.data_ptr(), _IT[t.dtype], n,
                                       float(scale), res.data_ptr(), _row_pitch(res), _stream_ptr(dev))
    _lib.check(st, "dl_embed_rows")
    return out if out is not None else res.view(*tokens.shape, W)


def embed_grad(grad: torch.Tensor, tokens: torch.Tensor, vocab: int, *, scale: float = 1.0, dtype: Optional[torch.dtype] = None,
               into: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient [vocab, width] of `embed_rows`: row v is `scale` times the sum of the rows of `grad` whose token is v.

    grad [*tokens.shape, width]; the rows of a token are summed in fp32 in ascending order and rounded once to `dtype` (that of
    `grad`, or fp32).  `into` [vocab, width] of that dtype: the sums are added to what it holds -- the gradient that a tied head
    has left there -- and only rows that some token names are touched; else the result is new and its other rows are zero.
    No atomics on floats: the same bits on every call."""
    _dev(grad, "grad")
    dev = grad.device
    t = _tokens_1d(tokens, dev)
    if grad.dim() < 1 or tuple(grad.shape[:-1]) != tuple(tokens.shape) and not (grad.dim() == 2 and grad.shape[0] == t.numel()):
        raise RuntimeError(f"grad must be [*tokens.shape, width]: got {tuple(grad.shape)} for tokens {tuple(tokens.shape)}")
    W, n = grad.shape[-1], t.numel()
    g = grad if grad.dim() == 2 else grad.reshape(n, W)
    if W > 1 and g.stride(1) != 1 or n > 1 and g.stride(0) < W:
        g = g.contiguous()
    _matrix(g, "grad")
    vocab = int(vocab)
    if vocab < 0:
        raise ValueError("vocab must not be negative")
    want = dtype if dtype is not None else (into.dtype if into is not None else g.dtype)
    if want not in (g.dtype, torch.float32):
        raise RuntimeError(f"the gradient of {g.dtype} rows is {g.dtype} or fp32, not {want}")
    if into is None:
        res = torch.empty((vocab, W), dtype=want, device=dev)
    else:
        res = into
        _dev(into, "into", dev)
        _matrix(into, "into")
        if tuple(into.shape) != (vocab, W) or into.dtype != want:
            raise RuntimeError(f"into must be a [{vocab}, {W}] {want} matrix")
        if _share_memory(into, g):
            raise RuntimeError("into must not share memory with grad")
    lib = _lib.load()
    ws_bytes = lib.dl_embed_grad_workspace_bytes(n, W)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    with _on(dev):
        st = lib.dl_embed_grad(g.data_ptr(), _DT[g.dtype], _row_pitch(g), n, W, t.data_ptr(), _IT[t.dtype], float(scale), int(into is not None),
                               res.data_ptr(), _DT[res.dtype], _row_pitch(res), vocab, ws.data_ptr() if ws is not None else 0, ws_bytes,
                               _stream_ptr(dev))
    _lib.check(st, "dl_embed_grad")
    return res


@torch.library.custom_op("distillery_amd::embed", mutates_args=())
def embed(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """`embed_rows` with autograd: differentiable with respect to `table` (a dense gradient, made by `embed_grad`), any number of times.
    A registered operator, as its backward is: torch.compile and FakeTensor tracing see through both."""
    return embed_rows(table, tokens, scale=scale)


@embed.register_fake
def _(table, tokens, scale=1.0):
    return table.new_empty((*tokens.shape, table.shape[1]))


# Its gradient as an operator of its own, so that a backward pass is traced as well (shapes alone) and differentiated again: linear in
# `grad`, with the lookup for its derivative.
@torch.library.custom_op("distillery_amd::embed_backward", mutates_args=())
def embed_backward_op(grad: torch.Tensor, tokens: torch.Tensor, vocab: int, scale: float) -> torch.Tensor:
    return embed_grad(grad, tokens, vocab, scale=scale)


@embed_backward_op.register_fake
def _(grad, tokens, vocab, scale):
    return grad.new_empty((vocab, grad.shape[-1]))


def _embed_setup(ctx, inputs, output):
    table, tokens, scale = inputs
    ctx.save_for_backward(tokens)
    ctx.vocab, ctx.scale = table.shape[0], scale


def _embed_backward(ctx, grad):
    (tokens,) = ctx.saved_tensors
    # Neither traced nor to be differentiated again: straight to the kernels (131 x 1024 fp32, forward and back: 115 us,
    # 142 through the dispatcher).
    if type(grad) is torch.Tensor and not torch.is_grad_enabled() and not is_in_torch_dispatch_mode():
        return embed_grad(grad, tokens, ctx.vocab, scale=ctx.scale), None, None
    return embed_backward_op(grad, tokens, ctx.vocab, ctx.scale), None, None


def _embed_backward_setup(ctx, inputs, output):
    _, tokens, _, scale = inputs
    ctx.save_for_backward(tokens)
    ctx.scale = scale


def _embed_twice(ctx, grad):
    (tokens,) = ctx.saved_tensors
    return embed(grad.contiguous(), tokens, ctx.scale), None, None, None


embed.register_autograd(_embed_backward, setup_context=_embed_setup)
embed_backward_op.register_autograd(_embed_twice, setup_context=_embed_backward_setup)
