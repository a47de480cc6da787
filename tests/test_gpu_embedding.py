"""GPU parity of the embedding lookup and its gradient against plain sums in float64."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
#: half a step of a type at 1 (the largest relative error of a rounding), and the smallest step
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
STEP = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.fixture(scope="module")
def D():
    import llm_distillery_amd as d
    d._lib.load()
    return d


def _tokens(n, vocab, seed, kind="text"):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((n,), vocab // 2)
    t = (torch.rand(n, generator=g).double().pow(4) * vocab).long().clamp_(max=vocab - 1)
    if kind == "padded":
        t = torch.where(torch.rand(n, generator=g) < 0.4, torch.tensor([-1, vocab, vocab + 7, -2 ** 31])[torch.randint(4, (n,), generator=g)], t)
    if kind == "none":
        t = torch.full((n,), -1)
    return t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 50, 7), (3, 100, 8), (131, 1000, 256), (2049, 300, 257), (5000, 777, 1032)])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_lookup_is_the_rounded_product(D, dtype, n, vocab, width, itype):
    g = torch.Generator().manual_seed(n)
    table = torch.randn(vocab, width, generator=g).to(dtype)
    t = _tokens(n, vocab, n, "padded").to(itype)
    scale = 11.3137085
    got = D.embed_rows(table.to(DEV), t.to(DEV), scale=scale).cpu()
    inside = (t >= 0) & (t < vocab)
    want = (table[torch.where(inside, t, torch.zeros_like(t)).long()].float() * torch.tensor(scale)).to(dtype)
    want[~inside] = 0
    assert torch.equal(got, want)


def test_lookup_keeps_shapes_strides_and_odd_addresses(D):
    g = torch.Generator().manual_seed(1)
    big = torch.randn(70, 131, generator=g).to(torch.bfloat16).to(DEV)
    table = big[:, 3:130]                                     # rows off every 16-byte boundary
    t = torch.randint(0, 70, (3, 5), generator=g).to(DEV)
    got = D.embed_rows(table, t)
    assert got.shape == (3, 5, 127) and torch.equal(got, table[t])
    out = torch.full((15, 200), 7.0, dtype=torch.bfloat16, device=DEV)
    D.embed_rows(table, t, out=out[:, 1:128])
    assert torch.equal(out[:, 1:128], table[t].view(15, 127)) and (out[:, :1] == 7).all() and (out[:, 128:] == 7).all()
    assert D.embed_rows(table, t[:0]).shape == (0, 5, 127)


def test_lookup_rows_beyond_32_bits_of_elements(D):
    table = torch.zeros((600000, 4096), dtype=torch.bfloat16, device=DEV)      # 2.46e9 elements
    table[599999] = 3.0
    table[0] = 1.0
    got = D.embed_rows(table, torch.tensor([599999, 0, 599998], device=DEV))
    assert (got[0] == 3).all() and (got[1] == 1).all() and (got[2] == 0).all()
    del table
    grad = D.embed_grad(torch.ones((2, 4096), dtype=torch.bfloat16, device=DEV), torch.tensor([599999, 5], device=DEV), 600000)
    assert (grad[599999] == 1).all() and (grad[5] == 1).all() and (grad[599998] == 0).all() and (grad[599000:599998] == 0).all()


def _grad_check(D, g, t, vocab, scale, into=None, dtype=None):
    n, width = g.shape
    want_type = dtype or (into.dtype if into is not None else g.dtype)
    inside = (t >= 0) & (t < vocab)
    ref = torch.zeros(vocab, width, dtype=torch.float64).index_add_(0, t[inside].long(), g[inside].double()) * float(np.float32(scale))
    mag = torch.zeros(vocab, width, dtype=torch.float64).index_add_(0, t[inside].long(), g[inside].double().abs()) * abs(scale)
    hits = torch.bincount(t[inside].long(), minlength=vocab).unsqueeze(1).double()
    old = into.double() if into is not None else torch.zeros_like(ref)
    ref = ref + old
    # every fp32 addition and the product (or the multiply-add) round once: 2^-24 of a partial sum of at most `mag`; then one
    # rounding to the gradient's type
    bound = (hits + 4) * 2.0 ** -24 * (mag + old.abs()) + HALF_ULP[want_type] * ref.abs() * (1 + 2.0 ** -10) + STEP[want_type]
    dev_into = into.to(DEV) if into is not None else None
    got = D.embed_grad(g.to(DEV), t.to(DEV), vocab, scale=scale, into=dev_into, dtype=dtype)
    assert got.dtype == want_type and got.shape == (vocab, width)
    err = (got.cpu().double() - ref).abs()
    assert (err <= bound).all(), f"worst ratio {(err / bound).max().item()}"
    untouched = hits[:, 0] == 0
    assert torch.equal(got.cpu()[untouched], (into if into is not None else torch.zeros(vocab, width, dtype=want_type))[untouched])
    if into is None:
        assert torch.equal(got, D.embed_grad(g.to(DEV), t.to(DEV), vocab, scale=scale, dtype=dtype))
    else:
        assert got is dev_into


@pytest.mark.parametrize("dtype,out", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, None), (torch.bfloat16, torch.float32),
                                       (torch.float16, torch.float32)])
@pytest.mark.parametrize("n,vocab,width,kind", [(1, 1, 1, "text"), (1, 50, 7, "text"), (33, 40, 64, "one"), (64, 3, 9, "padded"), (1024, 500, 40, "padded"),
                                                (1025, 500, 40, "padded"), (5000, 1500, 133, "text"), (4097, 2000, 24, "one"), (1500, 70, 16, "none")])
@pytest.mark.parametrize("add", [False, True])
def test_gradient(D, dtype, out, n, vocab, width, kind, add):
    gen = torch.Generator().manual_seed(n + width)
    g = torch.randn(n, width, generator=gen).to(dtype)
    into = torch.randn(vocab, width, generator=gen).to(out or dtype) if add else None
    _grad_check(D, g, _tokens(n, vocab, n, kind), vocab, 2.5, into=into, dtype=out)


@pytest.mark.parametrize("n,vocab", [(70000, 300000), (200000, 2_000_000)])
def test_gradient_of_long_lists_and_large_vocabularies(D, n, vocab):
    """More words than 64 workgroups of 2048, ids of two digits of 10 bits and of three of 7."""
    gen = torch.Generator().manual_seed(n)
    _grad_check(D, torch.randn(n, 5, generator=gen), _tokens(n, vocab, n, "padded"), vocab, 1.0)


def test_gradient_of_strided_rows_and_int32_tokens(D):
    gen = torch.Generator().manual_seed(5)
    big = torch.randn(300, 101, generator=gen).to(torch.bfloat16)
    t = _tokens(300, 90, 5).int()
    dense = D.embed_grad(big[:, 2:99].contiguous().to(DEV), t.to(DEV), 90, scale=0.5)
    holder = torch.zeros(90, 120, dtype=torch.bfloat16, device=DEV)
    got = D.embed_grad(big.to(DEV)[:, 2:99], t.to(DEV), 90, scale=0.5, into=holder[:, 5:102])
    assert torch.equal(got, dense) and (holder[:, :5] == 0).all() and (holder[:, 102:] == 0).all()
    three = D.embed_grad(big[:, 2:99].contiguous().view(3, 100, 97).to(DEV), t.view(3, 100).to(DEV), 90, scale=0.5)
    assert torch.equal(three, dense)


def test_gradient_without_tokens(D):
    g, t = torch.zeros((0, 12), device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV)
    assert (D.embed_grad(g, t, 30) == 0).all()
    into = torch.full((30, 12), 2.0, device=DEV)
    assert (D.embed_grad(g, t, 30, into=into) == 2).all()
    assert D.embed_grad(torch.zeros((4, 12), device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV), 0).shape == (0, 12)


def test_infinite_rows_reach_their_token_only(D):
    g = torch.ones(40, 16, dtype=torch.bfloat16)
    g[7] = float("inf")
    g[9] = float("nan")
    t = torch.arange(40) % 20
    t[30] = -1
    g[30] = float("nan")                                      # padding: never read into a sum
    got = D.embed_grad(g.to(DEV), t.to(DEV), 20).cpu()
    assert torch.isinf(got[7]).all() and torch.isnan(got[9]).all()
    rest = [v for v in range(20) if v not in (7, 9)]
    assert torch.isfinite(got[rest]).all() and (got[10] == 1).all() and (got[0] == 2).all()


def test_autograd_against_differences(D):
    gen = torch.Generator().manual_seed(9)
    table = torch.randn(50, 24, generator=gen).to(DEV).requires_grad_(True)
    t = _tokens(60, 50, 9, "padded").to(DEV).view(6, 10)
    w = torch.randn(6, 10, 24, generator=gen).to(DEV)
    loss = (D.embed(table, t, 3.0) * w).sum()
    loss.backward()
    direction = torch.randn(50, 24, generator=gen).to(DEV)
    with torch.no_grad():
        h = 2.0 ** -3                                         # linear: the difference has rounding only
        up, down = ((D.embed(table + s * h * direction, t, 3.0).double() * w.double()).sum() for s in (1, -1))
    slope = ((up - down) / (2 * h)).item()
    want = (table.grad.double() * direction.double()).sum().item()
    scale = (w.double().abs().sum() * 3 * (table.double().abs().max() + direction.double().abs().max())).item()
    assert abs(slope - want) <= 2.0 ** -22 / h * scale


def test_on_another_stream(D):
    gen = torch.Generator().manual_seed(3)
    g, t = torch.randn(3000, 64, generator=gen).to(DEV), _tokens(3000, 500, 3).to(DEV)
    here = D.embed_grad(g, t, 500)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        there = D.embed_grad(g, t, 500)
        rows = D.embed_rows(here, t)
    s.synchronize()
    assert torch.equal(here, there) and torch.equal(rows, here[t])


def test_refusals(D):
    table, t = torch.zeros(10, 8, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError):
        D.embed_rows(table.cpu(), t)
    with pytest.raises(RuntimeError):
        D.embed_rows(table, t.cpu())
    with pytest.raises(RuntimeError):
        D.embed_rows(table, t.float())
    with pytest.raises(RuntimeError):
        D.embed_rows(table.double(), t)
    with pytest.raises(RuntimeError):
        D.embed_rows(table.t(), t)
    with pytest.raises(RuntimeError):
        D.embed_rows(table, t, out=torch.zeros(2, 8, device=DEV))
    with pytest.raises(RuntimeError):
        D.embed_grad(torch.zeros(4, 8, device=DEV), t, 10)
    with pytest.raises(RuntimeError):
        D.embed_grad(torch.zeros(3, 8, device=DEV), t, 10, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        D.embed_grad(torch.zeros(3, 8, device=DEV), t, 10, into=torch.zeros(9, 8, device=DEV))
    with pytest.raises(ValueError):
        D.embed_grad(torch.zeros(3, 8, device=DEV), t, -1)
    lib = D._lib.load()
    g = torch.zeros(3, 8, device=DEV)
    args = [g.data_ptr(), 0, 8, 3, 8, t.data_ptr(), 1, 1.0, 0, table.data_ptr(), 0, 8, 10]
    assert lib.dl_embed_grad(*args, 0, 0, 0) == -7
    assert lib.dl_embed_grad(*args[:2], 7, *args[3:], 0, 0, 0) == -3
    assert lib.dl_embed_grad(g.data_ptr(), 0, 8, 3, 8, t.data_ptr(), 1, 1.0, 0, table.data_ptr(), 1, 8, 10, 0, 0, 0) == -2
    assert lib.dl_embed_rows(table.data_ptr(), 0, 8, 10, 8, t.data_ptr() + 4, 1, 3, 1.0, g.data_ptr(), 8, 0) == -6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_gradient_is_differentiated_again(D, dtype):
    """d/dw of <v, gradient of <w, embed(table)>> is embed(v); v comes dense and as one broadcast number."""
    gen = torch.Generator().manual_seed(21)
    table = torch.randn(50, 24, generator=gen).to(dtype).to(DEV).requires_grad_(True)
    t = _tokens(60, 50, 9, "padded").to(DEV).view(6, 10)
    w = torch.randn(6, 10, 24, generator=gen).to(dtype).to(DEV).requires_grad_(True)
    v = torch.randn(50, 24, generator=gen).to(dtype).to(DEV)
    grad, = torch.autograd.grad(D.embed(table, t, 3.0), table, w, create_graph=True)
    assert torch.equal(grad.detach(), D.embed_grad(w.detach(), t, 50, scale=3.0))
    again, = torch.autograd.grad(grad, w, v, retain_graph=True)
    assert torch.equal(again, D.embed_rows(v, t, scale=3.0))
    flat, = torch.autograd.grad(grad.sum(), w)
    assert torch.equal(flat, D.embed_rows(torch.ones_like(v), t, scale=3.0))


def test_registered_operators_and_a_compiled_step(D):
    gen = torch.Generator().manual_seed(22)
    table = torch.randn(40, 16, generator=gen).to(DEV).requires_grad_(True)
    t = _tokens(30, 40, 5, "padded").to(DEV).view(5, 6)
    w = torch.randn(5, 6, 16, generator=gen).to(DEV)
    from llm_distillery_amd import embedding
    torch.library.opcheck(embedding.embed, (table, t, 2.0))
    torch.library.opcheck(embedding.embed_backward_op, (w.clone().requires_grad_(True), t, 40, 2.0))
    step = lambda table, t, w: (D.embed(table, t, 2.0) * w).sum()  # noqa: E731
    want, = torch.autograd.grad(step(table, t, w), table)
    got, = torch.autograd.grad(torch.compile(step, backend="aot_eager", fullgraph=True)(table, t, w), table)
    assert torch.equal(got, want)


def test_a_traced_backward_pass_has_the_operator(D):
    from torch.fx.experimental.proxy_tensor import make_fx
    table = torch.randn(40, 16, device=DEV)
    t = _tokens(30, 40, 5, "padded").to(DEV)
    w = torch.randn(30, 16, device=DEV)

    def step(table, w):
        table = table.detach().requires_grad_(True)
        return torch.autograd.grad(D.embed(table, t, 2.0), table, w)[0]
    for mode in ("real", "fake"):
        graph = make_fx(step, tracing_mode=mode, _allow_non_fake_inputs=True)(table, w)
        assert any("embed_backward" in str(n.target) for n in graph.graph.nodes)
        assert torch.equal(graph(2 * table, 3 * w), step(2 * table, 3 * w))
