"""What a student needs to write its own continuations: sampling from its logits, and its head in 8-bit floating point or integers.  Thin
wrappers over the C ABI; all arithmetic runs in the HIP kernels."""
from __future__ import annotations

from typing import NamedTuple, Tuple, Union

import torch

from . import _lib
from .ops import _DT, _dev, _on, _row_pitch, _rows_2d, _stream_ptr


def _row_vector(t: torch.Tensor, n: int, dtype: torch.dtype, name: str, dev: torch.device) -> torch.Tensor:
    """`t`, one entry per row, as a contiguous vector."""
    if t.get_device() != dev.index or t.dtype != dtype or t.numel() != n:
        _dev(t, name, dev)
        raise RuntimeError(f"{name} must be a {dtype} tensor with one entry for each of the {n} rows")
    return t if t.is_contiguous() else t.contiguous()


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
    if V == 0:
        raise RuntimeError("the rows have no columns")
    u = _row_vector(u, R, torch.float32, "u", dev)
    T, k, p, m = temperature, top_k, top_p, min_p
    T_ptr = k_ptr = p_ptr = m_ptr = 0
    if isinstance(T, torch.Tensor):
        T = _row_vector(T, R, torch.float32, "temperature", dev)
        T_ptr = T.data_ptr()
    if isinstance(k, torch.Tensor):
        k = _row_vector(k, R, torch.int32, "top_k", dev)
        k_ptr = k.data_ptr()
    elif not 0 <= k <= 0x7fffffff:
        raise ValueError("top_k must not be negative")
    if isinstance(p, torch.Tensor):
        p = _row_vector(p, R, torch.float32, "top_p", dev)
        p_ptr = p.data_ptr()
    if isinstance(m, torch.Tensor):
        m = _row_vector(m, R, torch.float32, "min_p", dev)
        m_ptr = m.data_ptr()
    shape = logits.shape[:-1]
    tokens = torch.empty(shape, dtype=torch.int64, device=dev)
    logp = torch.empty(shape, dtype=torch.float32, device=dev)
    kept = torch.empty(shape, dtype=torch.int32, device=dev)
    with _on(dev):
        st = _lib.load().dl_sample_rows(x.data_ptr(), _DT[x.dtype], _row_pitch(x), R, V, u.data_ptr(), T_ptr, k_ptr, p_ptr, m_ptr,
                                        0.0 if T_ptr else float(T), 0 if k_ptr else int(k), 0.0 if p_ptr else float(p), 0.0 if m_ptr else float(m),
                                        tokens.data_ptr(), logp.data_ptr(), kept.data_ptr(), _stream_ptr(dev))
    _lib.check(st, "dl_sample_rows")
    return tokens, logp, kept


class BlockQuantized(NamedTuple):
    """A matrix [rows, width] held in 8-bit floating point (e4m3): `codes` [rows, width rounded up to whole blocks of 128] with zeros
    behind the last column, and `scales` fp32 [rows or row blocks of 128, column blocks]; an element is its code times its scale."""
    codes: torch.Tensor
    scales: torch.Tensor
    width: int

    def dequantize(self) -> torch.Tensor:
        """The matrix in fp32 (plain torch; for looking at it)."""
        rows = self.codes.shape[0]
        s = self.scales if self.scales.shape[0] == rows else self.scales.repeat_interleave(128, 0)[:rows]
        return (self.codes.float() * s.repeat_interleave(128, 1))[:, :self.width]


def _blocks(n: int) -> int:
    return -(-n // 128)


def quantize_blocks(x: torch.Tensor, *, rows: int = 1) -> BlockQuantized:
    """x [..., width] (bf16/fp16/fp32, rows evenly strided) in 8-bit floating point with one scale for every 128 values of a row
    (`rows` = 1: activations) or for every 128 x 128 values (`rows` = 128: weights, laid out once).

    A block's scale is its largest magnitude times 1 / 448 (in fp32), at least 2^-100; codes are the values over the scale, rounded to even."""
    _dev(x, "x")
    if rows not in (1, 128):
        raise ValueError("rows must be 1 or 128")
    v = x if x.dim() == 2 and x.stride(1) == 1 else _rows_2d(x if x.dim() > 1 else x.unsqueeze(0))
    if v.dtype not in _DT:
        raise RuntimeError("unsupported dtype")
    R, W = v.shape
    dev = v.device
    kb = _blocks(W)
    codes = torch.empty((R, kb * 128), dtype=torch.float8_e4m3fn, device=dev)
    if rows == 1:
        scales = torch.empty_strided((R, kb), (1, R), dtype=torch.float32, device=dev)      # the scales of a block of columns side by side
    else:
        scales = torch.empty((_blocks(R), kb), dtype=torch.float32, device=dev)
    if R and W:
        with _on(dev):
            st = _lib.load().dl_quantize_blocks(v.data_ptr(), _DT[v.dtype], _row_pitch(v), R, W, rows, codes.data_ptr(), kb * 128,
                                                scales.data_ptr(), scales.stride(0), scales.stride(1), _stream_ptr(dev))
        _lib.check(st, "dl_quantize_blocks")
    return BlockQuantized(codes, scales, W)


def _check_blocks(q: BlockQuantized, name: str, groups: int, blocks: int, dev: torch.device):
    """(address, row stride) of the codes and (address, strides) of the scales of an operand."""
    codes, scales = q.codes, q.scales
    if codes.device != dev or scales.device != dev:
        _dev(codes, f"{name}.codes", dev), _dev(scales, f"{name}.scales", dev)
    rows, wide = codes.shape
    pitch, one = codes.stride()
    if codes.dtype != torch.float8_e4m3fn or wide != blocks * 128 or rows and (one != 1 or rows > 1 and pitch < wide):
        raise RuntimeError(f"{name}.codes must be a float8_e4m3fn matrix of whole blocks of 128 columns, dense along its rows")
    if scales.dtype != torch.float32 or scales.shape != (groups, blocks):
        raise RuntimeError(f"{name}.scales must be fp32 [{groups}, {blocks}], not {tuple(scales.shape)}")
    return codes.data_ptr(), pitch if rows > 1 else wide, scales.data_ptr(), *scales.stride()


def matmul_blocks(a: BlockQuantized, b: BlockQuantized, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, width] times the transpose of b [N, width], both in 8-bit floating point: [M, N] in `dtype` (bf16/fp16/fp32).

    `a` has a scale for every 128 values of a row, `b` for every 128 x 128 (`quantize_blocks` with rows = 1 and 128).  A block's
    128 products are summed by the matrix unit, the scaled sums of the blocks in fp32, and the result is rounded once.  The matrix
    unit's sums are not fp32 sums: one is off by up to 2^-12 of the sum of its products' magnitudes (normal data: some 2e-5 of it),
    which fp32 results show.  A row's result has the same bits whatever rows it comes with."""
    dev = a.codes.device
    if dtype not in _DT:
        raise RuntimeError("unsupported dtype")
    if a.codes.dim() != 2 or b.codes.dim() != 2:
        raise RuntimeError("codes must be matrices")
    M, N, W = a.codes.shape[0], b.codes.shape[0], a.width
    if W != b.width:
        raise RuntimeError(f"a has {W} columns, b {b.width}")
    if W == 0:
        raise RuntimeError("the rows have no columns")
    _dev(a.codes, "a.codes")
    blocks = _blocks(W)
    left, right = _check_blocks(a, "a", M, blocks, dev), _check_blocks(b, "b", _blocks(N), blocks, dev)
    out = torch.empty((M, N), dtype=dtype, device=dev)
    if M and N:
        with _on(dev):
            st = _lib.load().dl_matmul_blocks(*left, M, *right, N, W, out.data_ptr(), _DT[dtype], N, _stream_ptr(dev))
        _lib.check(st, "dl_matmul_blocks")
    return out


class RowQuantized(NamedTuple):
    """A matrix [rows, width] held in 8-bit integers: `codes` int8 [rows, width rounded up to whole blocks of 128] with zeros behind the last
    column, and `scales` fp32 [rows]; an element is its code times its row's scale."""
    codes: torch.Tensor
    scales: torch.Tensor
    width: int

    def dequantize(self) -> torch.Tensor:
        """The matrix in fp32 (plain torch; for looking at it)."""
        return (self.codes.float() * self.scales.unsqueeze(1))[:, :self.width]


def quantize_rows(x: torch.Tensor) -> RowQuantized:
    """x [..., width] (bf16/fp16/fp32, rows evenly strided) in 8-bit integers with one scale for every row: a state, or the weights of an output
    channel (laid out once).

    A row's scale is its largest magnitude times 1 / 127 (in fp32), at least 2^-100; codes are the values over the scale, rounded to even, within
    [-127, 127].  A row with a NaN or an infinity has a scale of NaN."""
    _dev(x, "x")
    v = x if x.dim() == 2 and x.stride(1) == 1 else _rows_2d(x if x.dim() > 1 else x.unsqueeze(0))
    kind = _DT.get(v.dtype)
    if kind is None:
        raise RuntimeError("unsupported dtype")
    (R, W), pitch = v.shape, v.stride(0)
    if R <= 1:
        pitch = W
    elif pitch < W:
        raise RuntimeError("x: rows overlap; make them contiguous first")
    dev = v.device
    wide = (W + 127) // 128 * 128
    codes = v.new_empty(R, wide, dtype=torch.int8)
    scales = v.new_empty(R, dtype=torch.float32)
    if R:
        with _on(dev):
            st = _lib.load().dl_quantize_rows(v.data_ptr(), kind, pitch, R, W, codes.data_ptr(), wide, scales.data_ptr(), _stream_ptr(dev))
        if st:
            _lib.check(st, "dl_quantize_rows")
    return RowQuantized(codes, scales, W)


def _check_rows(codes: torch.Tensor, scales: torch.Tensor, name: str, wide: int, dev: torch.device):
    """(address, row stride) of the codes and the address of the scales of an operand, and how many rows it has."""
    here = dev.index
    if codes.get_device() != here or scales.get_device() != here:
        _dev(codes, f"{name}.codes", dev), _dev(scales, f"{name}.scales", dev)
    (rows, columns), (pitch, one) = codes.shape, codes.stride()
    if codes.dtype != torch.int8 or columns != wide or rows and (one != 1 or rows > 1 and pitch < wide):
        raise RuntimeError(f"{name}.codes must be an int8 matrix of whole blocks of 128 columns, dense along its rows")
    if scales.dtype != torch.float32 or scales.dim() != 1 or scales.numel() != rows or rows > 1 and not scales.is_contiguous():
        raise RuntimeError(f"{name}.scales must be a contiguous fp32 vector of {rows} entries")
    return codes.data_ptr(), pitch if rows > 1 else wide, scales.data_ptr(), rows


def matmul_rows(a: RowQuantized, b: RowQuantized, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, width] times the transpose of b [N, width], both in 8-bit integers with a scale for every row (`quantize_rows`): [M, N] in `dtype`
    (bf16/fp16/fp32).

    Sums of products are exact; a sum becomes a float, is multiplied with the product of the two scales (each rounded in fp32), and the result is
    rounded once.  A row's result has the same bits whatever rows it comes with.  Up to 130944 columns."""
    (a_codes, a_scales, W), (b_codes, b_scales, b_width), kind = a, b, _DT.get(dtype)
    if kind is None:
        raise RuntimeError("unsupported dtype")
    if a_codes.dim() != 2 or b_codes.dim() != 2:
        raise RuntimeError("codes must be matrices")
    if W != b_width:
        raise RuntimeError(f"a has {W} columns, b {b_width}")
    if W <= 0:
        raise RuntimeError("the rows have no columns")
    _dev(a_codes, "a.codes")
    dev, wide = a_codes.device, (W + 127) // 128 * 128
    *left, M = _check_rows(a_codes, a_scales, "a", wide, dev)
    *right, N = _check_rows(b_codes, b_scales, "b", wide, dev)
    out = a_codes.new_empty(M, N, dtype=dtype)
    if M and N:
        with _on(dev):
            st = _lib.load().dl_matmul_rows(*left, M, *right, N, W, out.data_ptr(), kind, N, _stream_ptr(dev))
        if st:
            _lib.check(st, "dl_matmul_rows")
    return out
