"""GPU parity of the 8-bit block quantisation (bit for bit) and of the matrix product over it (against float64)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def D():
    import llm_distillery_amd as d
    d._lib.load()
    return d


def e4m3(q):
    """The values of e4m3 nearest to q (fp32, at most 464 in magnitude), ties to the even code: by arithmetic."""
    q = q.double()
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -9))).clamp_min(-6.0) - 3.0)
    return torch.round(q / step) * step


def quantised(x, rows):
    """(code values [R, whole blocks] in float64, scales fp32) by the definition."""
    R, W = x.shape
    kb, g = -(-W // 128), -(-R // rows)
    full = torch.zeros(g * rows, kb * 128)
    full[:R, :W] = x.float()
    t = full.view(g, rows, kb, 128)
    scales = torch.maximum(t.abs().amax((1, 3)) * (torch.tensor(1.0) / torch.tensor(448.0)), torch.tensor(2.0 ** -100))
    return e4m3(t / scales[:, None, :, None]).view(g * rows, kb * 128)[:R], scales


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,W", [(1, 1), (1, 128), (3, 129), (5, 1000), (130, 257), (257, 2048)])
@pytest.mark.parametrize("rows", [1, 128])
def test_codes_and_scales_are_the_definition(D, dtype, R, W, rows):
    g = torch.Generator().manual_seed(W)
    x = (torch.randn(R, W, generator=g) * torch.exp(2 * torch.randn(R, W, generator=g))).to(dtype)
    x[0, : W // 2] = 0.0
    q = D.quantize_blocks(x.to(DEV), rows=rows)
    values, scales = quantised(x, rows)
    assert q.width == W and torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.codes.float().cpu().double(), values)
    assert torch.equal(q.dequantize().cpu(), (values.float() * scales.repeat_interleave(rows, 0)[:R].repeat_interleave(128, 1))[:, :W])


def test_zeros_tiny_values_views_and_shapes(D):
    x = torch.zeros(4, 300)
    x[1, 5] = 1e-42
    x[2, 7] = 2.0 ** -92
    q = D.quantize_blocks(x.to(DEV))
    values, scales = quantised(x, 1)
    assert torch.equal(q.codes.float().cpu().double(), values) and torch.equal(q.scales.cpu(), scales)
    g = torch.Generator().manual_seed(2)
    big = torch.randn(6, 333, generator=g).to(torch.bfloat16)
    part = D.quantize_blocks(big.to(DEV)[:, 3:332])
    whole = D.quantize_blocks(big[:, 3:332].contiguous().to(DEV))
    assert torch.equal(part.codes.view(torch.uint8), whole.codes.view(torch.uint8)) and torch.equal(part.scales, whole.scales)
    assert D.quantize_blocks(big.to(DEV).view(2, 3, 333)).codes.shape == (6, 384)
    assert D.quantize_blocks(big.to(DEV)[:0]).codes.shape == (0, 384)


def product(D, x, w, dtype, pitch=0):
    """The product through the kernels, and the float64 one of the same codes with the sums of magnitudes."""
    a, b = D.quantize_blocks(x.to(DEV)), D.quantize_blocks(w.to(DEV), rows=128)
    got = D.matmul_blocks(a, b, dtype=dtype)
    kb, N = a.scales.shape[1], w.shape[0]
    A = a.codes.float().cpu().double().view(-1, kb, 128) * a.scales.cpu().double().unsqueeze(2)
    B = b.codes.float().cpu().double().view(-1, kb, 128) * b.scales.cpu().double().repeat_interleave(128, 0)[:N].unsqueeze(2)
    A, B = A.view(x.shape[0], -1), B.view(N, -1)
    return got.cpu().double(), A @ B.t(), A.abs() @ B.abs().t()


def within(got, want, mag, blocks, dtype):
    # the matrix unit's sums are off by up to 2^-12 of the magnitudes; scaling and adding a block rounds twice in fp32; one
    # rounding to the result's type
    bound = (2.0 ** -12 + (blocks + 2) * 2.0 ** -23) * mag + torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + torch.finfo(dtype).tiny
    bad = (got - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} values off, worst ratio {((got - want).abs() / bound).max().item():.2f}"


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 48, 64, 65, 100, 129, 300])
@pytest.mark.parametrize("N,W", [(1, 128), (5, 40), (127, 300), (129, 128), (1000, 640), (517, 2500)])
def test_product(D, M, N, W):
    g = torch.Generator().manual_seed(M * 1000 + N)
    x = (torch.randn(M, W, generator=g) * torch.exp(torch.randn(1, W, generator=g))).to(torch.bfloat16)
    w = torch.randn(N, W, generator=g) * 0.02
    for dtype in (torch.float32, torch.bfloat16):
        got, want, mag = product(D, x, w, dtype)
        within(got, want, mag, -(-W // 128), dtype)


@pytest.mark.parametrize("M,N,W", [(700, 24000, 256), (4100, 4100, 384), (2049, 8200, 130), (260, 70001, 128)])
def test_large_tiles(D, M, N, W):
    g = torch.Generator().manual_seed(M)
    x, w = torch.randn(M, W, generator=g), torch.randn(N, W, generator=g)
    got, want, mag = product(D, x, w, torch.float16)
    within(got, want, mag, -(-W // 128), torch.float16)


@pytest.mark.parametrize("M", [3, 70, 2100])
def test_exact_where_every_sum_is(D, M):
    """Small whole numbers as values, scales of 1: every sum is exact in fp32, so the product is too, wherever an element lands."""
    g = torch.Generator().manual_seed(M)
    x = torch.randint(-4, 5, (M, 384), generator=g).float()
    w = torch.randint(-4, 5, (32 * 1025, 384), generator=g).float()
    x[:, ::128], w[:, ::128] = 448.0, 0.0                     # the largest magnitude of every block: scales of 1
    w[::128, ::128] = 448.0
    x[:, ::128] = torch.where(torch.rand(M, 1, generator=g) < 0.5, 448.0, -448.0)
    got = D.matmul_blocks(D.quantize_blocks(x.to(DEV)), D.quantize_blocks(w.to(DEV), rows=128), dtype=torch.float32)
    small = torch.arange(0, 32 * 1025, 7)                     # (448 * 448 * 3 + ... is a whole number below 2^24 as well)
    want = (x.double() @ w[small].double().t().contiguous()).float()
    diff = (got.cpu()[:, small] - want).abs()
    rows = (small % 128 != 0).nonzero()[:, 0]                 # without the 448s, where small products next to them may be cut off
    assert (diff[:, rows] == 0).all()


def test_rows_do_not_depend_on_their_neighbours(D):
    g = torch.Generator().manual_seed(8)
    x, w = torch.randn(2000, 1300, generator=g).to(DEV), torch.randn(9001, 1300, generator=g).to(DEV)
    b = D.quantize_blocks(w, rows=128)
    whole = D.matmul_blocks(D.quantize_blocks(x), b, dtype=torch.float32)
    for lo, hi in ((0, 1), (5, 21), (10, 50), (3, 200), (100, 900), (1000, 1016)):
        assert torch.equal(D.matmul_blocks(D.quantize_blocks(x[lo:hi]), b, dtype=torch.float32), whole[lo:hi])


@pytest.mark.parametrize("M", [4, 200])
def test_nan_and_infinity_stay_in_their_row(D, M):
    g = torch.Generator().manual_seed(9)
    x, w = torch.randn(M, 300, generator=g), torch.randn(500, 300, generator=g)
    x[1, 5], x[2, 299] = math.nan, math.inf
    got = D.matmul_blocks(D.quantize_blocks(x.to(DEV)), D.quantize_blocks(w.to(DEV), rows=128))
    assert torch.isnan(got[[1, 2]]).all() and torch.isfinite(got[0]).all() and torch.isfinite(got[3:]).all()


def test_views_of_codes_and_scales(D):
    g = torch.Generator().manual_seed(10)
    x, w = torch.randn(40, 256, generator=g).to(DEV), torch.randn(700, 256, generator=g).to(DEV)
    a, b = D.quantize_blocks(x), D.quantize_blocks(w, rows=128)
    want = D.matmul_blocks(a, b)
    holder = torch.zeros((700, 512), dtype=torch.uint8, device=DEV)
    holder[:, 128:384] = b.codes.view(torch.uint8)
    other = D.BlockQuantized(holder.view(torch.float8_e4m3fn)[:, 128:384], b.scales.t().contiguous().t(), 256)
    plain = D.BlockQuantized(a.codes, a.scales.contiguous(), 256)
    assert torch.equal(D.matmul_blocks(plain, other), want)
    assert torch.equal(D.matmul_blocks(D.BlockQuantized(a.codes[7:9], a.scales[7:9], 256), b), want[7:9])
    assert D.matmul_blocks(D.quantize_blocks(x[:0]), b).shape == (0, 700)


def test_addresses_beyond_32_bits(D):
    """Weights of more than 4 GiB, results of more than 2^31 elements."""
    b = D.BlockQuantized(torch.zeros((1_100_000, 4096), dtype=torch.float8_e4m3fn, device=DEV), torch.ones((8594, 32), device=DEV), 4096)
    b.codes.view(torch.uint8)[1_099_999] = 0x38               # 1.0
    x = torch.zeros((2100, 4096), device=DEV)
    x[-1], x[3] = 448.0, 448.0
    for rows in (slice(2096, 2100), slice(0, 2100)):
        got = D.matmul_blocks(D.quantize_blocks(x[rows]), b)
        assert got[-1, -1].item() == 448 * 4096 and (got[-1, :-1] == 0).all() and got[-2].abs().max().item() == 0
        del got


def test_refusals(D):
    x, w = torch.randn(4, 256, device=DEV), torch.randn(300, 256, device=DEV)
    a, b = D.quantize_blocks(x), D.quantize_blocks(w, rows=128)
    with pytest.raises(ValueError):
        D.quantize_blocks(x, rows=64)
    with pytest.raises(RuntimeError):
        D.quantize_blocks(x.cpu())
    with pytest.raises(RuntimeError):
        D.quantize_blocks(x.double())
    for p, q in ((a, D.quantize_blocks(w[:, :128], rows=128)), (a, D.quantize_blocks(w)), (b, b), (a._replace(codes=a.codes.view(torch.uint8)), b),
                 (a._replace(scales=a.scales.double()), b), (a._replace(scales=a.scales.cpu()), b), (a, b._replace(codes=b.codes[:, :128])),
                 (a._replace(width=100), b._replace(width=100))):
        with pytest.raises(RuntimeError):
            D.matmul_blocks(p, q)
    with pytest.raises(RuntimeError):
        D.matmul_blocks(a, b, dtype=torch.float64)
    lib = D._lib.load()
    c, s, o = b.codes.data_ptr(), b.scales.data_ptr(), torch.zeros(4, 300, device=DEV).data_ptr()
    assert lib.dl_matmul_blocks(c + 8, 256, s, 2, 1, 4, c, 256, s, 2, 1, 300, 256, o, 0, 300, 0) == -6
    assert lib.dl_matmul_blocks(c, 128, s, 2, 1, 4, c, 256, s, 2, 1, 300, 256, o, 0, 300, 0) == -3
    assert lib.dl_matmul_blocks(c, 256, 0, 2, 1, 4, c, 256, s, 2, 1, 300, 256, o, 0, 300, 0) == -1
    assert lib.dl_matmul_blocks(c, 256, s, 2, 1, 4, c, 256, s, 2, 1, 300, 256, o, 9, 300, 0) == -2
    assert lib.dl_quantize_blocks(x.data_ptr(), 0, 256, 4, 256, 2, c, 256, s, 2, 1, 0) == -3
