"""What the C entries of adjusted logits, integer products and clipped gradients refuse before any GPU work, and their shape-only forms."""
import ctypes
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import llm_distillery_amd as D  # noqa: E402

P = 4096                                                       # an address that is never used


def adjust(**kw):
    a = dict(logits=P, dtype=0, row_stride=100, n_rows=4, V=100, tokens=P, itype=0, token_stride=9, n_texts=4, length=9, token_rows=0, lengths=0, prompt=0,
             prompt_all=0, repetition=0, frequency=0, presence=0, repetition_all=1.0, frequency_all=0.0, presence_all=0.0, bias=0, bias_dtype=0, bias_stride=0,
             allowed=0, allowed_stride=0, n_masks=0, allowed_rows=0, out=P, out_stride=100, stream=0)
    assert set(kw) <= set(a)
    return D._lib.load().dl_adjust_rows(*{**a, **kw}.values())


def adjust_grad(**kw):
    a = dict(grad=P, dtype=0, grad_stride=100, logits=P, row_stride=100, n_rows=4, V=100, tokens=P, itype=0, token_stride=9, n_texts=4, length=9, token_rows=0,
             lengths=0, repetition=0, repetition_all=1.0, allowed=0, allowed_stride=0, n_masks=0, allowed_rows=0, out=P, out_stride=100, bias_grad=P, bias_dtype=0,
             workspace=P, workspace_bytes=1 << 20, stream=0)
    assert set(kw) <= set(a)
    return D._lib.load().dl_adjust_grad(*{**a, **kw}.values())


def test_adjusted_logits():
    assert adjust(dtype=3) == -2 and adjust(itype=2) == -2 and adjust(bias=P, bias_dtype=1) == -2
    assert adjust(row_stride=99) == -3 and adjust(out_stride=99) == -3 and adjust(n_rows=-1) == -3 and adjust(n_texts=2) == -3 and adjust(length=-1) == -3
    assert adjust(allowed=P, allowed_stride=3, n_masks=4) == -3 and adjust(allowed=P, allowed_stride=4, n_masks=3) == -3
    assert adjust(bias=P, bias_stride=99) == -3 and adjust(token_stride=-1) == -3
    assert adjust(V=1 << 31, row_stride=1 << 31, out_stride=1 << 31) == -4 and adjust(length=1 << 31, token_stride=1 << 31) == -4
    assert adjust(logits=P + 2) == -6 and adjust(out=P + 1, dtype=1) == -6 and adjust(tokens=P + 4, itype=1) == -6 and adjust(bias=P + 2) == -6
    assert adjust(allowed=P + 2, allowed_stride=4, n_masks=4) == -6
    assert adjust(logits=0) == -1 and adjust(out=0) == -1
    assert adjust(n_rows=0) == 0 and adjust(V=0) == 0


def test_their_gradient():
    assert adjust_grad(dtype=-1) == -2 and adjust_grad(bias_dtype=2) == -2
    assert adjust_grad(grad_stride=99) == -3 and adjust_grad(row_stride=1) == -3 and adjust_grad(out_stride=1) == -3
    assert adjust_grad(grad=0) == -1 and adjust_grad(logits=0) == -1
    assert adjust_grad(workspace=P + 8) == -6 and adjust_grad(grad=P + 1) == -6 and adjust_grad(bias_grad=P + 2) == -6
    need = D._lib.load().dl_adjust_grad_workspace_bytes(4, 100)
    assert need >= 400 and adjust_grad(workspace_bytes=need - 1) == -7 and adjust_grad(workspace=0) == -7
    assert D._lib.load().dl_adjust_grad_workspace_bytes(0, 100) == 0
    assert adjust_grad(V=0) == 0 and adjust_grad(n_rows=0, bias_grad=0) == 0


def test_texts_whose_last_place_is_beyond_32_bits():
    """The kernels count a text's places in 32 bits and step past its end by up to 8192: longer texts than 2^31 - 8192 are refused.  (Without logits: a
    call whose length is accepted is refused for them.)"""
    for length, status in ((2 ** 31 - 8192, -1), (2 ** 31 - 8191, -4), (2 ** 31 - 2048, -4), (2 ** 31 - 1, -4)):
        for itype in (0, 1):
            assert adjust(logits=0, itype=itype, n_texts=1, token_stride=length, length=length) == status
            assert adjust_grad(logits=0, itype=itype, n_texts=1, token_stride=length, length=length) == status


def test_integer_products():
    lib = D._lib.load()
    assert lib.dl_quantize_rows(P, 3, 256, 4, 256, P, 256, P, 0) == -2
    assert lib.dl_quantize_rows(P, 0, 255, 4, 256, P, 256, P, 0) == -3 and lib.dl_quantize_rows(P, 0, 256, 4, 250, P, 250, P, 0) == -3
    assert lib.dl_quantize_rows(0, 0, 256, 4, 256, P, 256, P, 0) == -1 and lib.dl_quantize_rows(P, 0, 256, 4, 256, P + 8, 256, P, 0) == -6
    assert lib.dl_quantize_rows(P, 0, 256, 4, 256, P, 264, P, 0) == -6 and lib.dl_quantize_rows(P, 0, 256, 0, 256, P, 256, P, 0) == 0
    mul = lambda a=P, sa=256, s=P, b=P, sb=256, K=256, out=P, dt=0, so=300: lib.dl_matmul_rows(a, sa, s, 4, b, sb, s, 300, K, out, dt, so, 0)  # noqa: E731
    assert mul(dt=9) == -2 and mul(sa=128) == -3 and mul(sb=240) == -3 and mul(K=0) == -3 and mul(so=299) == -3
    assert mul(a=0) == -1 and mul(s=0) == -1 and mul(out=0) == -1
    assert mul(a=P + 8) == -6 and mul(sa=264) == -6 and mul(out=P + 2) == -6 and mul(s=P + 2) == -6
    assert mul(K=130945, sa=131072, sb=131072) == -4


def test_rows_of_no_columns():
    lib = D._lib.load()
    assert lib.dl_quantize_rows(0, 0, 0, 4, 0, 0, 0, 0, 0) == -1 and lib.dl_quantize_rows(0, 0, 0, 0, 0, 0, 0, 0, 0) == 0      # (their scales are wanted)


def test_clipped_gradients():
    lib = D._lib.load()

    def call(at=(P, 2 * P), sizes=(100, 100), dtypes=(0, 1), scale=1.0, most=1.0, norm=P, given=0, ws=P, ws_bytes=1 << 20, clip=True):
        n = len(at)
        arrays = (ctypes.c_void_p * n)(*at), (ctypes.c_int64 * n)(*sizes), (ctypes.c_int32 * n)(*dtypes)
        if not clip:
            return lib.dl_grad_norm(*(ctypes.addressof(a) for a in arrays), n, scale, norm, ws, ws_bytes, 0)
        return lib.dl_clip_grads(*(ctypes.addressof(a) for a in arrays), n, scale, most, norm, given, ws, ws_bytes, 0)

    for clip in (True, False):
        assert call(dtypes=(0, 3), clip=clip) == -2 and call(sizes=(100, -1), clip=clip) == -3 and call(at=(P, 0), clip=clip) == -1
        assert call(at=(P, P + 1), clip=clip) == -6 and call(at=(P + 2, 2 * P), clip=clip) == -6 and call(norm=0, clip=clip) == -1
        assert call(norm=P + 2, clip=clip) == -6 and call(ws=P + 4, clip=clip) == -6 and call(ws=0, clip=clip) == -7 and call(ws_bytes=8, clip=clip) == -7
        for scale in (0.0, -1.0, math.inf, math.nan):
            assert call(scale=scale, clip=clip) == -3
        assert call(sizes=(1 << 62, 1), clip=clip) == -4 and call(at=(1 << 57, 2 * P), clip=clip) == -4
    assert call(most=-1.0) == -3 and call(most=math.nan) == -3
    assert call(at=(P, P + 396)) == -9 and call(at=(2 * P, P), sizes=(10, 2049)) == -9      # the last element of one, the first of the other
    assert b"overlap" in lib.dl_status_string(-9)
    sizes = (ctypes.c_int64 * 500)(*[1] * 500)
    need = [lib.dl_grad_norm_workspace_bytes(ctypes.addressof(sizes), n) for n in (0, 1, 240, 241, 500)]
    assert need[0] == 0 and need[1] == need[2] < need[3] < need[4]


def test_no_cpu_path():
    import pytest
    x = torch.randn(4, 64)
    for call in (lambda: D.adjust_rows(x), lambda: D.adjust_grad(x), lambda: D.adjust_logits(x), lambda: D.quantize_rows(x), lambda: D.grad_norm([x]),
                 lambda: D.clip_grads([x], 1.0)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_parameters_without_a_gradient_are_refused():
    import pytest
    for grads in ([None], [torch.ones(3), None], [], ()):
        with pytest.raises(RuntimeError, match="no gradients|must be tensors"):
            D.clip_grads(grads, 1.0)


def test_adjusted_logits_trace_with_fake_tensors_in_both_directions():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 6, 50, dtype=torch.bfloat16, requires_grad=True)
        tokens, words = torch.empty(12, 9, dtype=torch.int64), torch.empty(1, 2, dtype=torch.int32)
        weight = torch.empty(2, 6, 50, dtype=torch.bfloat16, requires_grad=True)
        for shape in ((50,), (2, 6, 50)):
            bias = torch.empty(shape, requires_grad=True)
            y = D.adjust_logits(x, tokens, bias=bias, repetition=1.5, allowed=words)
            assert y.shape == x.shape and y.dtype == torch.bfloat16
            gx, gb = torch.autograd.grad((y * weight).sum(), (x, bias), create_graph=True)
            assert gx.shape == x.shape and gx.dtype == torch.bfloat16 and gb.shape == shape and gb.dtype == torch.float32
            again, = torch.autograd.grad(gx.sum() + gb.sum(), weight)
            assert again.shape == weight.shape


def test_rows_without_columns_in_any_shape():
    """Their view is the one that rows with columns have: as many of them, none dropped."""
    for shape, rows in (((2, 3, 0), 6), ((4, 0), 4), ((0, 3, 0), 0), ((2, 0, 5), 0), ((2, 3, 5), 6)):
        assert D.ops._rows_2d(torch.empty(shape)).shape == (rows, shape[-1])
