"""GPU parity of the gradients' common norm and of clipping by it, against sums in float64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
STEP = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.fixture(scope="module")
def D():
    import llm_distillery_amd as d
    d._lib.load()
    return d


def some(sizes, seed, dtypes=(torch.float32, torch.bfloat16, torch.float16), std=0.1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=DEV) * std).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def exact_norm(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def near(norm, want):
    # fp64 sums of up to 2^30 exact squares in any order: far below the one rounding to fp32
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(norm.item() - want) <= 2.0 ** -24 * want * (1 + 2.0 ** -20) + 2.0 ** -149, (norm.item(), want)


def check_scaled(after, before, by):
    # the factor is rounded to fp32, the product in fp32, and to the type
    for a, b in zip(after, before):
        want = b.double() * by
        assert ((a.double() - want).abs() <= (2 * 2.0 ** -24 + HALF_ULP[b.dtype]) * want.abs() * (1 + 2.0 ** -20) + STEP[b.dtype]).all()


SIZES = [(1,), (3, 1, 7), (0, 5, 0), (8192, 8191, 8193, 1, 16384), (100003, 64, 1000000, 17), tuple(range(1, 300)), tuple([5] * 1000), (30_000_000, 3)]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("scale", [1.0, 2.5])
def test_norm_and_clipping(D, sizes, scale):
    grads = some(sizes, len(sizes))
    want = exact_norm(grads) * scale
    near(D.grad_norm(grads, scale=scale), want)
    for share in (0.25, 4.0):
        now = [g.clone() for g in grads]
        norm = D.clip_grads(now, want * share, scale=scale)
        near(norm, want)
        if share > 1 and scale == 1.0:
            assert all(torch.equal(a, b) for a, b in zip(now, grads))
        else:
            check_scaled(now, grads, scale * min(1.0, share))


def test_views_shapes_and_order_in_memory(D):
    """Parts of one buffer at every offset, transposed matrices, scalars, channels last."""
    g = torch.Generator(device=DEV).manual_seed(1)
    flat = torch.randn(200_000, generator=g, device=DEV).to(torch.bfloat16)
    image = torch.randn(2, 3, 4, 5, generator=g, device=DEV).to(memory_format=torch.channels_last)
    matrix, scalar = torch.randn(70, 90, generator=g, device=DEV), torch.randn((), generator=g, device=DEV)
    grads, at = [image, matrix.t(), scalar], 1
    for n in (1, 2, 3, 1000, 8192, 8193, 50001):
        grads.append(flat[at:at + n])
        at += n + 1
    before, rest = [v.clone() for v in grads], flat.clone()
    norm = D.clip_grads(grads, 1.0)
    want = exact_norm(before)
    near(norm, want)
    check_scaled(grads, before, 1.0 / want)
    touched = torch.zeros(200_000, dtype=torch.bool, device=DEV)
    at = 1
    for n in (1, 2, 3, 1000, 8192, 8193, 50001):
        touched[at:at + n] = True
        at += n + 1
    assert torch.equal(flat[~touched], rest[~touched])


def test_large_and_small_values(D):
    """Squares that leave the range of fp32 do not leave the sum's."""
    for v in (3e38, 1e25, 1e-25, 1e-45):
        grads = [torch.full((1000,), v, device=DEV), torch.zeros(10, device=DEV)]
        near(D.grad_norm(grads), min(exact_norm(grads), math.inf)) if v < 1e38 else None
    grads = [torch.full((1000,), 1e25, device=DEV)]
    D.clip_grads(grads, 1.0)
    assert torch.allclose(grads[0], torch.full((1000,), 1 / math.sqrt(1000), device=DEV), rtol=2.0 ** -22)
    zeros = [torch.zeros(100, device=DEV)]
    assert D.clip_grads(zeros, 0.0).item() == 0 and (zeros[0] == 0).all()
    ones = [torch.ones(100, device=DEV)]
    assert D.clip_grads(ones, 0.0).item() == 10 and (ones[0] == 0).all()      # nothing is allowed


@pytest.mark.parametrize("sizes", [(1000, 77), (40_000_001,)])
def test_the_one_rounding_is_the_results(D, sizes):
    """fp32 gradients by a factor of 64 bits: half a step of the result.  (What the factor, held in two floats, and the sum of the parts leave off
    is some 2^-46 of it; the sums of squares in 64 bits, pairwise here and there, agree to some 2^-48: together below 2^-24 * 2^-16.)"""
    grads = some(sizes, 9, (torch.float32,))
    for share, scale in ((0.3, 1.0), (1 / 7, 3.3), (2.0, 0.7)):
        scale = torch.tensor(scale).item()                    # (as fp32 has it)
        norm = exact_norm(grads) * scale
        most = torch.tensor(norm * share).item()
        now = [g.clone() for g in grads]
        D.clip_grads(now, most, scale=scale)
        for a, b in zip(now, grads):
            want = b.double() * (scale * min(1.0, most / norm))
            assert ((a.double() - want).abs() <= 2.0 ** -24 * want.abs() * (1 + 2.0 ** -16) + 2.0 ** -149).all()


@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
def test_a_norm_that_is_no_number_leaves_the_gradients(D, odd):
    grads = some((100, 20000, 3), 5)
    grads[1][19999] = odd
    before = [g.clone() for g in grads]
    norm = D.clip_grads(grads, 1.0, scale=2.0)
    assert math.isnan(norm.item()) if math.isnan(odd) else norm.item() == math.inf
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(grads, before))
    near(D.clip_grads(grads[2:], 1e9), exact_norm(grads[2:]))


@pytest.mark.parametrize("size", [4, 40_000_000])            # (with the sums added up in the launch that scales, and ahead of it)
def test_a_norm_beyond_fp32_leaves_the_gradients(D, size):
    """Finite gradients whose norm is infinite in fp32: nothing is written, as with any infinite norm."""
    grads = [torch.full((size,), 3e38, device=DEV)]
    before = grads[0].clone()
    assert D.grad_norm(grads).item() == math.inf
    assert D.clip_grads(grads, 1.0).item() == math.inf
    assert torch.equal(grads[0], before)


def test_a_norm_that_is_given(D):
    """Two halves of the gradients, as two cards have them, clipped by the norm of both; an infinite bound only scales."""
    grads = some((1000, 70000, 12, 400), 6)
    before = [g.clone() for g in grads]
    both = torch.stack([D.grad_norm(grads[:2], scale=3.0), D.grad_norm(grads[2:], scale=3.0)]).square().sum().sqrt()
    want = 3 * exact_norm(before)
    for part in (grads[:2], grads[2:]):
        assert D.clip_grads(part, 2.0, scale=3.0, norm=both) is both
    assert abs(both.item() - want) <= 2.0 ** -21 * want
    check_scaled(grads, before, 3 * 2.0 / both.item())
    now = [g.clone() for g in before]
    D.clip_grads(now, math.inf, scale=0.5)
    check_scaled(now, before, 0.5)


def test_the_same_bits_every_time_and_in_a_graph(D):
    grads = some((300_000, 77, 1_000_001), 7)
    before = [g.clone() for g in grads]
    norms = set()
    for _ in range(5):
        norms.add(D.grad_norm(grads).item())
    assert len(norms) == 1
    D.clip_grads(grads, 1.0)
    want = [g.clone() for g in grads]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = D.clip_grads(grads, 1.0)
    for k in range(4):
        for g, b in zip(grads, before):
            g.copy_(b * (k + 1))
        eager = [g.clone() for g in grads]
        eager_norm = D.clip_grads(eager, 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, eager_norm) and all(torch.equal(a, b) for a, b in zip(grads, eager))
        if k == 0:
            assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_another_stream(D):
    grads = some((100_000, 5), 8)
    want = exact_norm(grads)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm = D.clip_grads(grads, want / 2)
    s.synchronize()
    near(norm, want)
    assert abs(exact_norm(grads) - want / 2) <= 2.0 ** -8 * want


def test_parameters_of_a_module(D):
    """What a training loop does, against torch's own clipping (which divides by the norm plus 1e-6)."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(64, 200), torch.nn.GELU(), torch.nn.Linear(200, 10)).to(DEV)
    model(torch.randn(32, 64, device=DEV)).square().mean().backward()
    grads = [p.grad for p in model.parameters()]
    copies = [g.clone() for g in grads]
    norm = D.clip_grads((p.grad for p in model.parameters()), 0.01)
    for p, c in zip(model.parameters(), copies):
        p.grad = c
    want = torch.nn.utils.clip_grad_norm_(model.parameters(), 0.01)
    assert abs(norm.item() - want.item()) <= 2.0 ** -20 * want.item()
    for g, p in zip(grads, model.parameters()):
        assert torch.allclose(g, p.grad, rtol=2e-6 / want.item() + 2.0 ** -20, atol=0)


def test_more_than_2_31_elements(D):
    big = torch.zeros(2 ** 31 + 5000, dtype=torch.float16, device=DEV)
    big[-1], big[0], big[2 ** 31] = 3.0, 4.0, 12.0
    small = torch.full((1,), 84.0, device=DEV)
    assert D.clip_grads([big, small], 42.5).item() == 85.0
    assert big[-1].item() == 1.5 and big[0].item() == 2.0 and big[2 ** 31].item() == 6.0 and small.item() == 42.0


def test_refusals(D):
    a = torch.ones(100, device=DEV)
    for call in (lambda: D.grad_norm([]), lambda: D.grad_norm([a.cpu()]), lambda: D.grad_norm([a, a.cpu()]), lambda: D.grad_norm([a.double()]),
                 lambda: D.grad_norm([a[::2]]), lambda: D.grad_norm([a[:1].expand(5)]), lambda: D.grad_norm([a.view(10, 10)[:, :5]]),
                 lambda: D.grad_norm([a.to_sparse()]), lambda: D.clip_grads([a, a], 1.0), lambda: D.clip_grads([a[:60], a[59:]], 1.0),
                 lambda: D.clip_grads([a], 1.0, norm=a), lambda: D.clip_grads([a], 1.0, norm=torch.ones((), device=DEV, dtype=torch.float64)),
                 lambda: D.clip_grads([a], 1.0, norm=torch.ones(()))):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: D.clip_grads([a], -1.0), lambda: D.clip_grads([a], math.nan), lambda: D.clip_grads([a], 1.0, scale=0.0), lambda: D.grad_norm([a], scale=-1.0),
                 lambda: D.grad_norm([a], scale=math.inf), lambda: D.grad_norm([a], scale=math.nan)):
        with pytest.raises(ValueError):
            call()
    assert (a == 1).all()
    near(D.grad_norm([a, a]), math.sqrt(200))                 # only read: the same one twice counts twice


def test_autograd_sees_that_gradients_are_clipped(D):
    """Gradients that are to be differentiated again and were clipped in between: an error, no derivative of what they were not."""
    w = torch.randn(50, generator=torch.Generator(device=DEV).manual_seed(10), device=DEV).requires_grad_()
    grad, = torch.autograd.grad(w.pow(3).sum(), w, create_graph=True)
    z, parts = grad.square().sum(), torch.ones(30, device=DEV)
    D.grad_norm([grad])
    assert grad._version == 0
    D.clip_grads([grad, parts[:10], parts[10:]], 1e-3)
    assert grad._version == 1 and parts._version == 2
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def check_rounded_once(after, before, by):
    """By a factor of 64 bits: half a step of an fp32 result (what the norm and the factor leave off is below 2^-16 of that, as above); half a
    step of a type of 16 bits behind that of the fp32 number that it is rounded from."""
    for a, b in zip(after, before):
        want = b.double() * by
        half = 2.0 ** -24 if b.dtype == torch.float32 else 2.0 ** -24 * (1 + 2.0 ** -7) + HALF_ULP[b.dtype]
        assert ((a.double() - want).abs() <= half * want.abs() * (1 + 2.0 ** -16) + STEP[b.dtype]).all()


@pytest.mark.parametrize("most", [1.0, 1e-6, 3e-38])
def test_factors_smaller_than_fp32_holds(D, most):
    """Norms above 1e38: the factor is subnormal or 0 in fp32, the results are not."""
    most, given = torch.tensor(most).item(), torch.tensor(2e38, device=DEV)
    grads = some((1001, 12, 70_000), 11, (torch.float32, torch.bfloat16), std=4e35)
    norm = exact_norm(grads)
    assert 0.9e38 < norm < 3e38
    for kw, by in (({}, most / norm), (dict(norm=given), most / given.item())):
        now = [g.clone() for g in grads]
        D.clip_grads(now, most, **kw)
        check_rounded_once(now, grads, by)


def test_one_rounding_at_any_offset_and_in_any_number(D):
    """Three tables of tensors of all types and of odd sizes, parts of one buffer, a norm that is given."""
    grads = some((*range(1, 600), 100_003, 64, 1_000_000, 17), 12)
    flat, = some((90_001,), 13, (torch.float32,))
    grads += [flat[1:4], flat[5:50_000], flat[50_002:]]
    norm = exact_norm(grads)
    most = torch.tensor(norm / 3).item()
    for kw, by in (({}, most / norm), (dict(norm=torch.tensor(7.0, device=DEV), scale=0.75), 0.75 * min(1.0, most / 7.0))):
        now = [g.clone() for g in grads[:-3]]
        whole = flat.clone()
        now += [whole[1:4], whole[5:50_000], whole[50_002:]]
        D.clip_grads(now, most, **kw)
        check_rounded_once(now, grads, by)
        assert whole[0] == flat[0] and whole[4] == flat[4] and torch.equal(whole[50_000:50_002], flat[50_000:50_002])
