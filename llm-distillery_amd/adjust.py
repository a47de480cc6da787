"""Logits made ready for the sampler -- penalties for what a text has already, biases, masks of allowed tokens -- and the gradient of
that.  Thin wrappers over the C ABI; all arithmetic runs in the HIP kernels."""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd.graph import increment_version
from torch.utils._python_dispatch import is_in_torch_dispatch_mode

from . import _lib
from .ops import _DT, _IT, _dev, _on, _rows_2d, _share_memory, _stream_ptr
from .rollout import _row_vector

Number = Union[float, torch.Tensor]


def _logit_rows(t: torch.Tensor, name: str, dev: Optional[torch.device] = None) -> torch.Tensor:
    """t [..., V] as [rows, V] without a copy."""
    if dev is None or t.get_device() != dev.index:
        _dev(t, name, dev)
    if t.dtype not in _DT:
        raise RuntimeError(f"{name}: unsupported dtype")
    x = t if t.dim() == 2 and t.stride(1) == 1 else _rows_2d(t if t.dim() > 1 else t.unsqueeze(0))
    (R, V), pitch = x.shape, x.stride(0)
    if pitch < V and R > 1:
        raise RuntimeError(f"{name}: rows overlap; make them contiguous first")
    return x


def _check_repetition(v: float) -> None:
    """Of a number for all rows: what the kernels take is its fp32 form, which is 0 below half the smallest subnormal."""
    if not 2.0 ** -149 <= v <= 3.0e38:
        raise ValueError("repetition must be positive and finite in fp32")


def _per_row(v: Number, rows: int, name: str, dev: torch.device) -> Tuple[Optional[torch.Tensor], float]:
    """A setting as (one fp32 entry per row, 0) or (nothing, the number for all)."""
    return (_row_vector(v, rows, torch.float32, name, dev), 0.0) if isinstance(v, torch.Tensor) else (None, float(v))


def _texts(tokens: Optional[torch.Tensor], token_rows: Optional[torch.Tensor], rows: int, dev: torch.device) -> Tuple[tuple, tuple]:
    """The texts as the C ABI takes them -- address, index type, stride, number, length, address of the map -- and what has to stay alive."""
    if tokens is None:
        if token_rows is not None:
            raise RuntimeError("token_rows without tokens")
        return (0, 0, 0, 0, 0, 0), ()
    if tokens.get_device() != dev.index:
        _dev(tokens, "tokens", dev)
    kind, t = _IT.get(tokens.dtype), tokens
    if kind is None:
        raise RuntimeError("tokens must be int32 or int64")
    if t.dim() != 2:
        if t.dim() == 0:
            raise RuntimeError("tokens must be [..., length]")
        t = t.unsqueeze(0) if t.dim() == 1 else t.flatten(0, -2)
    (n, length), (pitch, one) = t.shape, t.stride()
    if one != 1 and length > 1:
        t, pitch = t.contiguous(), length
    if token_rows is not None:
        token_rows = _row_vector(token_rows, rows, torch.int32, "token_rows", dev)
    elif n not in (1, rows):
        raise RuntimeError(f"{n} texts for {rows} rows and no token_rows")
    return (t.data_ptr(), kind, pitch if n > 1 else length, n, length, token_rows.data_ptr() if token_rows is not None else 0), (t, token_rows)


def _masks(allowed: Optional[torch.Tensor], allowed_rows: Optional[torch.Tensor], rows: int, V: int, dev: torch.device) -> Tuple[tuple, tuple]:
    """The masks the same way: address, stride, number, address of the map."""
    if allowed is None:
        if allowed_rows is not None:
            raise RuntimeError("allowed_rows without allowed")
        return (0, 0, 0, 0), ()
    if allowed.get_device() != dev.index:
        _dev(allowed, "allowed", dev)
    words = -(-V // 32)
    m = allowed if allowed.dim() != 1 else allowed.unsqueeze(0)
    if m.dtype != torch.int32 or m.dim() < 2 or m.shape[-1] < words:
        raise RuntimeError(f"allowed must be int32 [masks, {words}], one bit for each of the {V} tokens")
    if m.dim() > 2:
        m = m.flatten(0, -2)
    (n, held), (pitch, one) = m.shape, m.stride()
    if one != 1 and held > 1 or pitch < words and n > 1:
        m, pitch = m.contiguous(), held
    if allowed_rows is not None:
        allowed_rows = _row_vector(allowed_rows, rows, torch.int32, "allowed_rows", dev)
    elif n not in (1, rows):
        raise RuntimeError(f"{n} masks for {rows} rows and no allowed_rows")
    return (m.data_ptr(), pitch if n > 1 else held, n, allowed_rows.data_ptr() if allowed_rows is not None else 0), (m, allowed_rows)


def _written(out: Optional[torch.Tensor], x: torch.Tensor, name: str, over: str, others: tuple = ()) -> torch.Tensor:
    """The matrix that the result goes to: new, or `out` checked -- `x` itself, or memory that neither `x` nor `others` have."""
    if out is None:
        return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient and the call records none: detach it, or call under torch.no_grad()")
    R, V = x.shape
    o = _logit_rows(out, name, x.device)
    if tuple(o.shape) != (R, V) or o.dtype != x.dtype:
        raise RuntimeError(f"{name} must be a [{R}, {V}] {x.dtype} matrix")
    same = o.data_ptr() == x.data_ptr() and (R <= 1 or o.stride(0) == x.stride(0))
    if not same and _share_memory(o, x) or any(_share_memory(o, t) for t in others):
        raise RuntimeError(f"{name} must be {over} itself or share no memory with the arguments")
    return o


def adjust_rows(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, token_rows: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, prompt: Union[int, torch.Tensor] = 0, repetition: Number = 1.0, frequency: Number = 0.0,
                presence: Number = 0.0, bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                allowed_rows: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Logits [..., V] (bf16/fp16/fp32, rows evenly strided) with penalties, a bias and a mask, in this order:

        x / `repetition` (positive x) or x * `repetition` for every token of the row's text, prompt and all;
        minus `frequency` times how often the text has the token behind the prompt, minus `presence` where it has it there;
        plus `bias`;  -inf where the row's mask does not allow the token.

    tokens: int32/int64 [..., length], a text for each row, or one for all, or any number of which row r has number `token_rows`[r] (int32;
    negative: none).  Ids outside [0, V) are padding.  A row has the first `lengths`[r] entries (int32; None: all), the first `prompt` (a
    number, or int32 per row) of which are its prompt's.  Each penalty is a number or an fp32 tensor with one entry per row; `repetition` is
    positive.
    bias: [V] for all rows or [..., V], fp32 or of the logits' dtype.
    allowed: int32 words, bit v % 32 of word v // 32 for token v, [masks, words]: a mask for each row, or one for all, or any number of which
    row r has number `allowed_rows`[r] (int32; negative: every token is allowed).  A masked token is -inf whatever its logit was; a row whose mask
    allows nothing is -inf throughout, and `sample_rows` gives it token -1.

    Arithmetic is fp32, rounded once to the logits' dtype.  Returns a new tensor, or `out`, which may be the logits themselves.  Autograd knows of the
    write into `out`: a backward pass that needs what was there raises.  `out` must not require a gradient unless recording is off."""
    x = _logit_rows(logits, "logits")
    R, V = x.shape
    dev = x.device
    (text, alive), (mask, alive_too) = _texts(tokens, token_rows, R, dev), _masks(allowed, allowed_rows, R, V, dev)
    if lengths is not None:
        lengths = _row_vector(lengths, R, torch.int32, "lengths", dev)
    prompt_rows, prompt_all = (_row_vector(prompt, R, torch.int32, "prompt", dev), 0) if isinstance(prompt, torch.Tensor) else (None, int(prompt))
    rep, rep_all = (None, repetition) if type(repetition) is float else _per_row(repetition, R, "repetition", dev)
    freq, freq_all = (None, frequency) if type(frequency) is float else _per_row(frequency, R, "frequency", dev)
    pres, pres_all = (None, presence) if type(presence) is float else _per_row(presence, R, "presence", dev)
    if rep is None:
        _check_repetition(rep_all)
    b_ptr = b_dtype = b_stride = 0
    others = ()
    if bias is not None:
        if bias.get_device() != dev.index:
            _dev(bias, "bias", dev)
        if bias.dtype not in (torch.float32, x.dtype):
            raise RuntimeError(f"bias must be fp32 or {x.dtype}")
        b = bias if bias.dim() == 1 else _logit_rows(bias, "bias", dev)
        if b.shape[-1] != V or b.dim() == 2 and b.shape[0] not in (1, R):
            raise RuntimeError(f"bias must be [{V}] or [{R}, {V}]")
        if b.dim() == 1 and V > 1 and b.stride(0) != 1:
            b = b.contiguous()
        b_ptr, b_dtype, b_stride = b.data_ptr(), _DT[b.dtype], b.stride(0) if b.dim() == 2 and b.shape[0] > 1 else 0
        others = (b if b.dim() == 2 else b.unsqueeze(0),)
    res = _written(out, x, "out", "the logits", others)
    with _on(dev):
        st = _lib.load().dl_adjust_rows(x.data_ptr(), _DT[x.dtype], x.stride(0) if R > 1 else V, R, V, *text, 0 if lengths is None else lengths.data_ptr(),
                                        0 if prompt_rows is None else prompt_rows.data_ptr(), prompt_all, 0 if rep is None else rep.data_ptr(),
                                        0 if freq is None else freq.data_ptr(), 0 if pres is None else pres.data_ptr(), rep_all, freq_all, pres_all,
                                        b_ptr, b_dtype, b_stride, *mask, res.data_ptr(), res.stride(0) if R > 1 else V, _stream_ptr(dev))
    if st:
        _lib.check(st, "dl_adjust_rows")
    if out is not None:
        increment_version(out)
    return out if out is not None else res if logits.dim() == 2 else res.view(logits.shape)


def adjust_grad(grad: torch.Tensor, logits: Optional[torch.Tensor] = None, tokens: Optional[torch.Tensor] = None, *,
                token_rows: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, repetition: Number = 1.0,
                allowed: Optional[torch.Tensor] = None, allowed_rows: Optional[torch.Tensor] = None, want_logits: bool = True,
                want_bias: bool = False, bias_dtype: torch.dtype = torch.float32,
                out: Optional[torch.Tensor] = None) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """The gradients of `adjust_rows` by its logits and by a bias [V] that all rows share, from that by its result, `grad` [..., V].

    By the logits: `grad` over or times `repetition` at the tokens of the row's text (by the sign of the `logits`, which are of the dtype of
    `grad` and not needed without tokens), 0 where the mask does not allow the token, whatever `grad` has there.  By the bias: the sum of the rows of
    `grad` over what their masks allow, fp32 or in the dtype of `grad`, in an order that does not change between calls.  (A bias of each row's own has
    the gradient that the logits have without tokens.)  Texts, masks and `repetition` as for `adjust_rows`.  `out`, for the first, may be
    `grad` itself (and is written as by `adjust_rows`).  Returns (by the logits or None, by the bias or None)."""
    g = _logit_rows(grad, "grad")
    R, V = g.shape
    dev = g.device
    (text, alive), (mask, alive_too) = _texts(tokens, token_rows, R, dev), _masks(allowed, allowed_rows, R, V, dev)
    if lengths is not None:
        lengths = _row_vector(lengths, R, torch.int32, "lengths", dev)
    rep, rep_all = (None, repetition) if type(repetition) is float else _per_row(repetition, R, "repetition", dev)
    if rep is None:
        _check_repetition(rep_all)
    if bias_dtype not in (torch.float32, g.dtype):
        raise RuntimeError(f"the bias's gradient is fp32 or {g.dtype}")
    x = None
    if logits is not None:
        x = _logit_rows(logits, "logits", dev)
        if x.shape != g.shape or x.dtype != g.dtype:
            raise RuntimeError(f"logits must be [{R}, {V}] {g.dtype} as grad is")
    elif tokens is not None and want_logits:
        raise RuntimeError("the gradient by the logits needs them where there are tokens")
    if out is not None and not want_logits:
        raise RuntimeError("out without want_logits")
    res = _written(out, g, "out", "grad", () if x is None else (x,)) if want_logits else None
    lib = _lib.load()
    by_bias = torch.empty(V, dtype=bias_dtype, device=dev) if want_bias else None
    ws_bytes = lib.dl_adjust_grad_workspace_bytes(R, V) if want_bias else 0
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    with _on(dev):
        st = lib.dl_adjust_grad(g.data_ptr(), _DT[g.dtype], g.stride(0) if R > 1 else V, 0 if x is None else x.data_ptr(),
                                0 if x is None else x.stride(0) if R > 1 else V, R, V, *text, 0 if lengths is None else lengths.data_ptr(),
                                0 if rep is None else rep.data_ptr(), rep_all, *mask, 0 if res is None else res.data_ptr(),
                                0 if res is None else res.stride(0) if R > 1 else V, 0 if by_bias is None else by_bias.data_ptr(),
                                _DT[bias_dtype], 0 if ws is None else ws.data_ptr(), ws_bytes, _stream_ptr(dev))
    if st:
        _lib.check(st, "dl_adjust_grad")
    if out is not None:
        increment_version(out)
    return (out if out is not None else res if not want_logits or grad.dim() == 2 else res.view(grad.shape)), by_bias


# ---- autograd.  Registered operators with shape-only forms, so that torch.compile and FakeTensor tracing see through both directions.  The two
# gradients are linear in `grad`, and each other's and their own derivatives: a backward pass is differentiated again, any number of times.

def _either(rows: Optional[torch.Tensor], number):
    return number if rows is None else rows


@torch.library.custom_op("distillery_amd::adjust", mutates_args=())
def adjust_op(logits: torch.Tensor, bias: Optional[torch.Tensor], tokens: Optional[torch.Tensor], token_rows: Optional[torch.Tensor],
              lengths: Optional[torch.Tensor], allowed: Optional[torch.Tensor], allowed_rows: Optional[torch.Tensor],
              prompt_rows: Optional[torch.Tensor], prompt: int, repetition_rows: Optional[torch.Tensor], repetition: float,
              frequency_rows: Optional[torch.Tensor], frequency: float, presence_rows: Optional[torch.Tensor], presence: float) -> torch.Tensor:
    return adjust_rows(logits, tokens, token_rows=token_rows, lengths=lengths, prompt=_either(prompt_rows, prompt),
                       repetition=_either(repetition_rows, repetition), frequency=_either(frequency_rows, frequency),
                       presence=_either(presence_rows, presence), bias=bias, allowed=allowed, allowed_rows=allowed_rows)


@adjust_op.register_fake
def _(logits, *rest):
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


@torch.library.custom_op("distillery_amd::adjust_backward", mutates_args=())
def adjust_backward_op(grad: torch.Tensor, logits: Optional[torch.Tensor], tokens: Optional[torch.Tensor], token_rows: Optional[torch.Tensor],
                       lengths: Optional[torch.Tensor], allowed: Optional[torch.Tensor], allowed_rows: Optional[torch.Tensor],
                       repetition_rows: Optional[torch.Tensor], repetition: float) -> torch.Tensor:
    return adjust_grad(grad, logits, tokens, token_rows=token_rows, lengths=lengths, repetition=_either(repetition_rows, repetition), allowed=allowed,
                       allowed_rows=allowed_rows)[0]


@adjust_backward_op.register_fake
def _(grad, *rest):
    return torch.empty(grad.shape, dtype=grad.dtype, device=grad.device)


@torch.library.custom_op("distillery_amd::adjust_bias_backward", mutates_args=())
def adjust_bias_backward_op(grad: torch.Tensor, allowed: Optional[torch.Tensor], allowed_rows: Optional[torch.Tensor], dtype: torch.dtype) -> torch.Tensor:
    return adjust_grad(grad, allowed=allowed, allowed_rows=allowed_rows, want_logits=False, want_bias=True, bias_dtype=dtype)[1]


@adjust_bias_backward_op.register_fake
def _(grad, allowed, allowed_rows, dtype):
    return torch.empty(grad.shape[-1:], dtype=dtype, device=grad.device)


def _even(grad: torch.Tensor) -> torch.Tensor:
    """A gradient as autograd hands it down, expanded or transposed as it may be, with rows as the kernels take them."""
    if not grad.is_contiguous():
        s, n = grad.stride(), grad.shape
        lead = all(n[d] == 1 or s[d] == s[-2] * math.prod(n[d + 1:-1]) for d in range(grad.dim() - 1))
        if grad.dim() < 2 or s[-1] != 1 or not lead or s[-2] < n[-1]:
            return grad.contiguous()
    return grad


def _adjust_setup(ctx, inputs, output):
    logits, bias, tokens, token_rows, lengths, allowed, allowed_rows, _, _, repetition_rows, repetition = inputs[:11]
    if repetition_rows is None and repetition == 1.0:
        tokens = None                                         # the text multiplied with nothing
    text = (logits, tokens, token_rows, lengths) if tokens is not None else (None,) * 4
    ctx.save_for_backward(*text, allowed, allowed_rows, repetition_rows if tokens is not None else None)
    ctx.repetition = repetition if tokens is not None else 1.0
    ctx.bias = None if bias is None else (bias.shape, bias.dtype)


def _adjust_backward(ctx, grad):
    logits, tokens, token_rows, lengths, allowed, allowed_rows, repetition_rows = ctx.saved_tensors
    want_logits, want_bias = ctx.needs_input_grad[0], ctx.bias is not None and ctx.needs_input_grad[1]
    by_logits = by_bias = None
    grad = _even(grad)
    shared = want_bias and ctx.bias[0].numel() == grad.shape[-1]
    if shared and type(grad) is torch.Tensor and not torch.is_grad_enabled() and not is_in_torch_dispatch_mode():
        # Neither traced nor to be differentiated again: both in one sweep.
        by_logits, by_bias = adjust_grad(grad, logits, tokens, token_rows=token_rows, lengths=lengths, repetition=_either(repetition_rows, ctx.repetition),
                                         allowed=allowed, allowed_rows=allowed_rows, want_logits=want_logits, want_bias=True,
                                         bias_dtype=ctx.bias[1])
        return (by_logits, by_bias.view(ctx.bias[0])) + (None,) * 13
    if want_logits:
        by_logits = adjust_backward_op(grad, logits, tokens, token_rows, lengths, allowed, allowed_rows, repetition_rows, ctx.repetition)
    if shared:
        by_bias = adjust_bias_backward_op(grad, allowed, allowed_rows, ctx.bias[1]).view(ctx.bias[0])
    elif want_bias:                                           # of each row's own
        by_bias = adjust_backward_op(grad, None, None, None, None, allowed, allowed_rows, None, 1.0).to(ctx.bias[1]).view(ctx.bias[0])
    return (by_logits, by_bias) + (None,) * 13


def _adjust_backward_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[1:8])
    ctx.repetition = inputs[8]


def _adjust_twice(ctx, grad):
    return (adjust_backward_op(grad.contiguous(), *ctx.saved_tensors, ctx.repetition),) + (None,) * 8


def _bias_backward_setup(ctx, inputs, output):
    grad, allowed, allowed_rows, _ = inputs
    ctx.save_for_backward(allowed, allowed_rows)
    ctx.like = grad.shape, grad.dtype


def _bias_twice(ctx, grad):
    allowed, allowed_rows = ctx.saved_tensors
    rows = grad.to(ctx.like[1]).expand(ctx.like[0]).contiguous()
    return adjust_backward_op(rows, None, None, None, None, allowed, allowed_rows, None, 1.0), None, None, None


adjust_op.register_autograd(_adjust_backward, setup_context=_adjust_setup)
adjust_backward_op.register_autograd(_adjust_twice, setup_context=_adjust_backward_setup)
adjust_bias_backward_op.register_autograd(_bias_twice, setup_context=_bias_backward_setup)


def adjust_logits(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, token_rows: Optional[torch.Tensor] = None,
                  lengths: Optional[torch.Tensor] = None, prompt: Union[int, torch.Tensor] = 0, repetition: Number = 1.0, frequency: Number = 0.0,
                  presence: Number = 0.0, bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                  allowed_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`adjust_rows` with autograd, for losses on the distribution that a text was drawn from: differentiable with respect to `logits` and `bias`, any
    number of times (penalties and their settings are constants).  Its gradients are `adjust_grad`'s."""
    rows = lambda v: v if isinstance(v, torch.Tensor) else None  # noqa: E731
    number = lambda v, kind: kind(0) if isinstance(v, torch.Tensor) else kind(v)  # noqa: E731
    return adjust_op(logits, bias, tokens, token_rows, lengths, allowed, allowed_rows, rows(prompt), number(prompt, int), rows(repetition),
                     number(repetition, float), rows(frequency), number(frequency, float), rows(presence), number(presence, float))
