"""GPU parity of the 8-bit integer quantisation (bit for bit) and of the matrix product over it (exact sums)."""
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


def quantised(x):
    """(codes [R, whole blocks], scales) by the definition, each operation in fp32."""
    R, W = x.shape
    x = x.float()
    scales = torch.maximum(x.abs().amax(1) * (torch.tensor(1.0) / torch.tensor(127.0)), torch.tensor(2.0 ** -100))
    codes = torch.zeros(R, -(-W // 128) * 128, dtype=torch.int8)
    codes[:, :W] = torch.round(x / scales.unsqueeze(1)).clamp(-127, 127).to(torch.int8)
    return codes, scales


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,W", [(1, 1), (1, 128), (3, 129), (5, 1000), (130, 257), (257, 2048), (3, 4096), (7, 5001), (2, 16385), (3, 40000)])
def test_codes_and_scales_are_the_definition(D, dtype, R, W):
    g = torch.Generator().manual_seed(W)
    x = (torch.randn(R, W, generator=g) * torch.exp(torch.randn(R, W, generator=g))).to(dtype)
    x[0, : W // 2] = 0.0
    q = D.quantize_rows(x.to(DEV))
    codes, scales = quantised(x)
    assert q.width == W and torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    assert torch.equal(q.dequantize().cpu(), (codes.float() * scales.unsqueeze(1))[:, :W])


def test_zeros_tiny_values_ties_views_and_shapes(D):
    x = torch.zeros(4, 300)
    x[1, 5] = 1e-42
    x[2, 7] = 2.0 ** -92
    x[3, :6] = torch.tensor([127.0, 0.5, 1.5, -0.5, -2.5, -127.0])      # scale 1 (127 * fl(1 / 127) is 1): ties go to even
    q = D.quantize_rows(x.to(DEV))
    codes, scales = quantised(x)
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
    g = torch.Generator().manual_seed(2)
    big = torch.randn(6, 333, generator=g).to(torch.bfloat16)
    part, whole = D.quantize_rows(big.to(DEV)[:, 3:332]), D.quantize_rows(big[:, 3:332].contiguous().to(DEV))
    assert torch.equal(part.codes, whole.codes) and torch.equal(part.scales, whole.scales)
    assert D.quantize_rows(big.to(DEV).view(2, 3, 333)).codes.shape == (6, 384) and D.quantize_rows(big.to(DEV)[0]).codes.shape == (1, 384)
    assert D.quantize_rows(big.to(DEV)[:0]).codes.shape == (0, 384)


def codes(R, W, seed, most=127):
    """Any codes, in whole blocks with zeros behind the last column, and scales."""
    g = torch.Generator().manual_seed(seed)
    c = torch.zeros(R, -(-W // 128) * 128, dtype=torch.int8)
    c[:, :W] = torch.randint(-most, most + 1, (R, W), generator=g)
    return c, torch.exp(torch.randn(R, generator=g)) * 0.01


def product(D, a, b, W, dtype):
    """The kernels' product, and the sums and scales that it is to be made of."""
    A, B = (D.RowQuantized(c.to(DEV), s.to(DEV), W) for c, s in (a, b))
    got = D.matmul_rows(A, B, dtype=dtype).cpu()
    sums = a[0].double() @ b[0].double().t().contiguous()     # whole numbers below 2^31: exact
    return got, sums.float() * (a[1].unsqueeze(1) * b[1].unsqueeze(0))


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 48, 64, 65, 100, 129, 300])
@pytest.mark.parametrize("N,W", [(1, 128), (5, 40), (127, 300), (129, 128), (1000, 640), (517, 2500), (64, 1)])
def test_product_bit_for_bit(D, M, N, W):
    a, b = codes(M, W, M * 1000 + N), codes(N, W, N)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got, want = product(D, a, b, W, dtype)
        assert torch.equal(got, want.to(dtype))


@pytest.mark.parametrize("M,N,W", [(700, 24000, 256), (4100, 4100, 384), (2049, 8200, 130), (260, 70001, 128), (1025, 1025, 4000), (8200, 300, 512)])
def test_large_tiles_bit_for_bit(D, M, N, W):
    a, b = codes(M, W, M), codes(N, W, N)
    got, want = product(D, a, b, W, torch.float16)
    assert torch.equal(got, want.half())


@pytest.mark.parametrize("M,N,W", [(61, 32896, 128), (61, 50257, 256), (1, 65664, 130), (33, 20011, 300), (8, 14337, 128), (130, 9001, 640), (64, 4099, 1000), (299, 5391, 257)])
def test_even_small_tiles_bit_for_bit(D, M, N, W):
    """Small tiles of fewer columns than they have room for, several a compute unit."""
    a, b = codes(M, W, M), codes(N, W, N)
    for dtype in (torch.float32, torch.bfloat16):
        got, want = product(D, a, b, W, dtype)
        assert torch.equal(got, want.to(dtype))


@pytest.mark.parametrize("M,N", [(1, 7), (40, 200), (300, 300)])
def test_the_largest_sums(D, M, N):
    """The widest rows of the largest codes, -128 among them: sums of up to 2^31 - 2^21."""
    W = 130944
    a, b = torch.full((M, W), -128, dtype=torch.int8), torch.full((N, W), -128, dtype=torch.int8)
    b[-1] = 127
    one = torch.ones
    got, want = product(D, (a, one(M)), (b, one(N)), W, torch.float32)
    assert torch.equal(got, want) and want[0, 0] == 128.0 * 128 * W


def test_quantised_product_is_near_the_real_one(D):
    """Codes are off by half a step of their row's scale each (and the scale's rounding): the products' sum by what that allows."""
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(50, 1000, generator=g), torch.randn(300, 1000, generator=g) * 0.02
    a, b = D.quantize_rows(x.to(DEV)), D.quantize_rows(w.to(DEV))
    got = D.matmul_rows(a, b, dtype=torch.float32).cpu().double()
    sa, sb = a.scales.cpu().double().unsqueeze(1), b.scales.cpu().double()
    bound = 0.5001 * (sa * w.double().abs().sum(1) + x.double().abs().sum(1, keepdim=True) * sb + 0.5001 * 1000 * sa * sb)
    assert ((got - x.double() @ w.double().t()).abs() <= bound).all()


def test_rows_do_not_depend_on_their_neighbours(D):
    a, b = codes(2000, 1300, 8), codes(9001, 1300, 9)
    B = D.RowQuantized(b[0].to(DEV), b[1].to(DEV), 1300)
    ac, sc = a[0].to(DEV), a[1].to(DEV)
    whole = D.matmul_rows(D.RowQuantized(ac, sc, 1300), B, dtype=torch.float32)
    for lo, hi in ((0, 1), (5, 21), (10, 50), (3, 200), (100, 900), (1000, 1016)):
        assert torch.equal(D.matmul_rows(D.RowQuantized(ac[lo:hi], sc[lo:hi], 1300), B, dtype=torch.float32), whole[lo:hi])


@pytest.mark.parametrize("M", [4, 200])
def test_nan_and_infinity_stay_in_their_row(D, M):
    g = torch.Generator().manual_seed(9)
    x, w = torch.randn(M, 300, generator=g), torch.randn(500, 300, generator=g)
    x[1, 5], x[2, 299] = math.nan, -math.inf
    q = D.quantize_rows(x.to(DEV))
    assert torch.isnan(q.scales[1:3]).all() and torch.isfinite(q.scales[3:]).all() and (q.codes[1:3] == 0).all()
    got = D.matmul_rows(q, D.quantize_rows(w.to(DEV)))
    assert torch.isnan(got[[1, 2]]).all() and torch.isfinite(got[0]).all() and torch.isfinite(got[3:]).all()


def test_views_of_codes_and_scales(D):
    a, b = codes(40, 256, 10), codes(700, 256, 11)
    A, B = (D.RowQuantized(c.to(DEV), s.to(DEV), 256) for c, s in (a, b))
    want = D.matmul_rows(A, B)
    holder = torch.ones((700, 512), dtype=torch.int8, device=DEV)
    holder[:, 128:384] = B.codes
    assert torch.equal(D.matmul_rows(A, D.RowQuantized(holder[:, 128:384], B.scales, 256)), want)
    assert torch.equal(D.matmul_rows(D.RowQuantized(A.codes[7:9], A.scales[7:9], 256), B), want[7:9])
    assert torch.equal(D.matmul_rows(A, D.RowQuantized(B.codes[3:500], B.scales[3:500], 256)), want[:, 3:500])
    assert D.matmul_rows(D.quantize_rows(torch.randn(0, 256, device=DEV)), B).shape == (0, 700)


def test_addresses_beyond_32_bits(D):
    """Weights of more than 4 GiB, results of more than 2^31 elements."""
    b = D.RowQuantized(torch.zeros((1_100_000, 4096), dtype=torch.int8, device=DEV), torch.ones(1_100_000, device=DEV), 4096)
    b.codes[1_099_999] = 1
    x = torch.zeros((2100, 4096), device=DEV)
    x[-1], x[3] = 127.0, 127.0
    for rows in (slice(2096, 2100), slice(0, 2100)):
        got = D.matmul_rows(D.quantize_rows(x[rows]), b, dtype=torch.float32 if rows.start else torch.bfloat16)
        assert got[-1, -1].item() == torch.tensor(127.0 * 4096).to(got.dtype).item() and (got[-1, :-1] == 0).all() and got[-2].abs().max().item() == 0
        del got


def test_captured_and_on_another_stream(D):
    g = torch.Generator(device=DEV).manual_seed(12)
    x, b = torch.randn(33, 500, generator=g, device=DEV), D.quantize_rows(torch.randn(900, 500, generator=g, device=DEV))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = D.matmul_rows(D.quantize_rows(x), b)
    s.synchronize()
    assert torch.equal(other, D.matmul_rows(D.quantize_rows(x), b))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = D.matmul_rows(D.quantize_rows(x), b)
    for _ in range(4):
        x.normal_(generator=g)
        want = D.matmul_rows(D.quantize_rows(x), b).clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_refusals(D):
    x, w = torch.randn(4, 256, device=DEV), torch.randn(300, 256, device=DEV)
    a, b = D.quantize_rows(x), D.quantize_rows(w)
    for call in (lambda: D.quantize_rows(x.cpu()), lambda: D.quantize_rows(x.double()), lambda: D.quantize_rows(x[:1].expand(4, 256))):
        with pytest.raises(RuntimeError):
            call()
    for p, q in ((a, D.quantize_rows(w[:, :128])), (a._replace(codes=a.codes.view(torch.uint8)), b), (a._replace(scales=a.scales.double()), b),
                 (a._replace(scales=a.scales.cpu()), b), (a, b._replace(codes=b.codes[:, :128])), (a._replace(width=100), b._replace(width=100)),
                 (a, b._replace(scales=b.scales[:299])), (a, b._replace(scales=torch.ones(600, device=DEV)[::2])), (a._replace(width=0), b._replace(width=0)),
                 (a._replace(codes=a.codes.t()), b), (a._replace(codes=a.codes[0]), b)):
        with pytest.raises(RuntimeError):
            D.matmul_rows(p, q)
    with pytest.raises(RuntimeError):
        D.matmul_rows(a, b, dtype=torch.float64)
    wide = torch.zeros(2, 130944 + 128, dtype=torch.int8, device=DEV)
    with pytest.raises(RuntimeError):
        D.matmul_rows(*[D.RowQuantized(wide, torch.ones(2, device=DEV), 130944 + 1)] * 2)


def test_more_rows_than_a_launch_takes(D):
    n = 33_488_896 + 77
    g = torch.Generator(device=DEV).manual_seed(13)
    x = torch.randn((n, 3), generator=g, device=DEV, dtype=torch.bfloat16)
    q = D.quantize_rows(x)
    for rows in (slice(0, 2 ** 18), slice(33_488_896 - 2 ** 18, n)):
        some = D.quantize_rows(x[rows])
        assert torch.equal(q.codes[rows], some.codes) and torch.equal(q.scales[rows], some.scales)
    assert torch.equal(some.scales.cpu(), quantised(x[rows].cpu())[1])


def test_rows_of_no_columns_have_the_least_scale(D):
    """As rows of zeros have it, and no memory as it was found."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        found = torch.full((5,), math.nan, device=DEV)
        del found                                             # (what the scales are likely to get)
        q = D.quantize_rows(torch.empty(5, 0, dtype=dtype, device=DEV))
        assert q.codes.shape == (5, 0) and q.width == 0 and (q.scales == 2.0 ** -100).all()
        assert torch.equal(q.scales, D.quantize_rows(torch.zeros(5, 3, dtype=dtype, device=DEV)).scales)
