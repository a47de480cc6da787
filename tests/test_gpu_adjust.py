"""GPU parity of adjusted logits (penalties, biases, masks) and their gradient against the definition in float64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
STEP = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def D():
    import llm_distillery_amd as d
    d._lib.load()
    return d


def bits(allowed):
    """Truth values [masks, V] as int32 words."""
    n, V = allowed.shape
    words = -(-V // 32)
    full = torch.zeros(n, words * 32, dtype=torch.int64)
    full[:, :V] = allowed.long()
    return (full.view(n, words, 32) << torch.arange(32)).sum(2).to(torch.int32)      # (bit 31: the conversion wraps)


def texts(n, length, V, seed, padded=True):
    """Ids as text has them, some of them padding."""
    g = torch.Generator().manual_seed(seed)
    t = (torch.rand(n, length, generator=g).double().pow(4) * V).long().clamp_(max=V - 1)
    if padded and length:
        t = torch.where(torch.rand(n, length, generator=g) < 0.2, torch.tensor([-1, V, V + 5, -2 ** 31])[torch.randint(4, (n, length), generator=g)], t)
    return t


def per_row(v, r):
    """A setting of row r as the kernels see it: an fp32 number."""
    return float((v[r] if isinstance(v, torch.Tensor) else torch.tensor(v, dtype=torch.float32)))


def said(V, r, tokens, token_rows, lengths, prompt):
    """(how often behind the prompt, whether at all) of row r's text."""
    count, seen = torch.zeros(V, dtype=torch.float64), torch.zeros(V, dtype=torch.bool)
    if tokens is None:
        return count, seen
    t = int(token_rows[r]) if token_rows is not None else 0 if tokens.shape[0] == 1 else r
    if not 0 <= t < tokens.shape[0]:
        return count, seen
    n = tokens.shape[1] if lengths is None else max(0, min(int(lengths[r]), tokens.shape[1]))
    p = int(prompt[r]) if isinstance(prompt, torch.Tensor) else prompt
    for i, v in enumerate(tokens[t, :n].tolist()):
        if 0 <= v < V:
            seen[v] = True
            count[v] += i >= p
    return count, seen


def mask_of(V, r, allowed, allowed_rows):
    if allowed is None:
        return torch.ones(V, dtype=torch.bool)
    m = int(allowed_rows[r]) if allowed_rows is not None else 0 if allowed.shape[0] == 1 else r
    return allowed[m] if 0 <= m < allowed.shape[0] else torch.ones(V, dtype=torch.bool)


def expected(x, tokens=None, token_rows=None, lengths=None, prompt=0, repetition=1.0, frequency=0.0, presence=0.0, bias=None, allowed=None,
             allowed_rows=None):
    """The result in float64, and the sum of the magnitudes that it is made from."""
    R, V = x.shape
    y, size = torch.empty(R, V, dtype=torch.float64), torch.empty(R, V, dtype=torch.float64)
    for r in range(R):
        count, seen = said(V, r, tokens, token_rows, lengths, prompt)
        z = x[r].double()
        rep, freq, pres = (per_row(v, r) for v in (repetition, frequency, presence))
        z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
        less = torch.where(count > 0, freq * count + pres, 0.0)
        b = torch.zeros(V, dtype=torch.float64) if bias is None else (bias if bias.dim() == 1 else bias[min(r, bias.shape[0] - 1)]).double()
        y[r] = torch.where(mask_of(V, r, allowed, allowed_rows), z - less + b, -math.inf)
        size[r] = z.abs() + torch.where(count > 0, abs(freq) * count + abs(pres), 0.0) + b.abs()
    return y, size


def check(got, want, size, dtype):
    # in fp32 at most six roundings (the penalty's product or quotient, frequency times count, plus presence, less that, plus bias), each at
    # most 2^-24 of a value that is no larger than the magnitudes' sum; then one to the type
    got, size = got.double().cpu(), torch.where(size.isfinite(), size, 0.0)
    odd = ~want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[odd & ~want.isnan()], want[odd & ~want.isnan()])
    bound = 6 * 2.0 ** -24 * size * (1 + 2.0 ** -20) + HALF_ULP[dtype] * want.abs() * (1 + 2.0 ** -20) + STEP[dtype]
    bad = ((got - want).abs() > bound) & ~odd
    assert not bad.any(), f"{int(bad.sum())} values off, worst ratio {((got - want).abs() / bound)[~odd].max().item():.2f}"


def on(v):
    return v.to(DEV) if isinstance(v, torch.Tensor) else v


def settings(R, seed):
    g = torch.Generator().manual_seed(seed)
    pick = lambda *v: torch.tensor(v)[torch.randint(len(v), (R,), generator=g)]  # noqa: E731
    return {"repetition": pick(1.0, 1.3, 0.8), "frequency": pick(0.0, 0.5, -0.25), "presence": pick(0.0, 0.7, -0.1)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
@pytest.mark.parametrize("R,V,L", [(1, 1, 1), (2, 7, 3), (3, 33, 0), (5, 1000, 64), (9, 4099, 300), (4, 40000, 2500), (17, 8192, 1)])
def test_everything_together(D, dtype, itype, R, V, L):
    g = torch.Generator().manual_seed(R * V)
    x = (torch.randn(R, V, generator=g) * 3).to(dtype)
    t = texts(R, L, V, V).to(itype)
    lengths = torch.randint(-1, L + 3, (R,), generator=g).int()
    prompt = torch.randint(0, L + 2, (R,), generator=g).int()
    allowed = torch.rand(R, V, generator=g) < 0.6
    bias = torch.randn(V, generator=g)
    s = settings(R, V)
    got = D.adjust_rows(x.to(DEV), t.to(DEV), lengths=lengths.to(DEV), prompt=prompt.to(DEV), bias=bias.to(DEV), allowed=bits(allowed).to(DEV),
                        **{k: on(v) for k, v in s.items()})
    check(got, *expected(x, t, None, lengths, prompt, bias=bias, allowed=allowed, **s), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["repetition", "frequency", "presence", "bias", "bias_rows", "bias_one_row", "bias_half", "allowed", "nothing"])
def test_each_alone(D, dtype, which):
    R, V, L = 6, 2311, 150
    g = torch.Generator().manual_seed(7)
    x = (torch.randn(R, V, generator=g) * 3).to(dtype)
    t = texts(R, L, V, 8)
    kw = {"repetition": {"repetition": 1.7}, "frequency": {"frequency": 0.3}, "presence": {"presence": -1.5}, "bias": {"bias": torch.randn(V, generator=g)},
          "bias_rows": {"bias": torch.randn(R, V, generator=g)}, "bias_one_row": {"bias": torch.randn(1, V, generator=g)},
          "bias_half": {"bias": torch.randn(V, generator=g).to(dtype)}, "allowed": {"allowed": torch.rand(1, V, generator=g) < 0.02}, "nothing": {}}[which]
    call = {k: bits(v).to(DEV) if k == "allowed" else on(v) for k, v in kw.items()}
    got = D.adjust_rows(x.to(DEV), t.to(DEV), **call)
    check(got, *expected(x, t, **kw), dtype)
    if which == "nothing":
        assert torch.equal(got.cpu(), x)
    if which in ("bias", "allowed"):
        assert torch.equal(D.adjust_rows(x.to(DEV), **call), got)      # no text


def test_maps_of_texts_and_masks(D):
    """Rows of one conversation with more and more of it, others, none, in any order; masks shared, and none."""
    R, V = 40, 5000
    g = torch.Generator().manual_seed(9)
    x = torch.randn(R, V, generator=g)
    t = texts(3, 77, V, 10)
    token_rows = torch.tensor([0] * 15 + [2, 1, 2, -1, 3, 2 ** 30] + [1] * 10 + [0] * 9).int()
    lengths = torch.tensor(list(range(15)) + [5, 70, 4, 9, 9, 9] + list(range(77, 67, -1)) + [3, 3, 77, 78, 0, 1, 20, 5, 6]).int()
    prompt = torch.tensor([2] * 8 + [5] * 7 + [0] * 25).int()
    allowed = torch.rand(4, V, generator=g) < 0.5
    allowed_rows = torch.randint(-1, 5, (R,), generator=g).int()
    s = settings(R, 11)
    got = D.adjust_rows(x.to(DEV), t.to(DEV), token_rows=token_rows.to(DEV), lengths=lengths.to(DEV), prompt=prompt.to(DEV), allowed=bits(allowed).to(DEV),
                        allowed_rows=allowed_rows.to(DEV), **{k: on(v) for k, v in s.items()})
    check(got, *expected(x, t, token_rows, lengths, prompt, allowed=allowed, allowed_rows=allowed_rows, **s), torch.float32)


def test_a_token_many_times_and_long_texts(D):
    """Counts beyond half a word, of one token and of all."""
    V = 300
    x = torch.full((3, V), 8.0)
    t = torch.full((3, 70000), 5)
    t[1, 1::2] = 299
    t[2] = torch.arange(70000) % V
    kw = {"frequency": 2.0 ** -10, "presence": 0.5, "repetition": 2.0, "prompt": 3}
    for length in (70000, 40000, 32768, 32767, 100):
        lengths = torch.full((3,), length).int()
        got = D.adjust_rows(x.to(DEV), t.to(DEV), lengths=lengths.to(DEV), **kw)
        check(got, *expected(x, t, None, lengths, **kw), torch.float32)
    short = t[:, :32767].contiguous()                        # the most that half a word counts
    check(D.adjust_rows(x.to(DEV), short.to(DEV), **kw), *expected(x, short, **kw), torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan(D, dtype):
    V = 600
    x = torch.zeros(3, V)
    x[:, 0:6] = torch.tensor([math.inf, -math.inf, math.nan, -0.0, torch.finfo(dtype).max, torch.finfo(dtype).min])
    x[1] = -math.inf
    x = x.to(dtype)
    t = torch.arange(6).repeat(3, 1)
    allowed = torch.ones(3, V, dtype=torch.bool)
    allowed[2, :7] = False
    bias = torch.zeros(V)
    bias[9], bias[10] = -math.inf, math.nan
    allowed[0, 10] = False
    kw = {"repetition": 1.25, "presence": 1.0, "bias": bias}
    got = D.adjust_rows(x.to(DEV), t.to(DEV), allowed=bits(allowed).to(DEV), **{k: on(v) for k, v in kw.items()}).cpu()
    want, size = expected(x, t, allowed=allowed, **kw)
    want = torch.where(want.abs() > torch.finfo(dtype).max * (1 + HALF_ULP[dtype] / 2), want.sign() * math.inf, want)
    check(got, want, size, dtype)
    assert torch.isneginf(got[2, :7]).all() and torch.isneginf(got[0, 9]) and torch.isneginf(got[0, 10]) and torch.isnan(got[2, 10])


def test_a_mask_that_leaves_nothing_gives_the_sampler_nothing(D):
    x = torch.randn(3, 1000, device=DEV)
    allowed = torch.zeros(2, 1000, dtype=torch.bool)
    allowed[1, 999] = True
    y = D.adjust_rows(x, allowed=bits(allowed).to(DEV), allowed_rows=torch.tensor([0, 1, -1], dtype=torch.int32, device=DEV))
    token, logp, kept = D.sample_rows(y, torch.tensor([0.5, 0.5, 0.5], device=DEV))
    assert token[:2].tolist() == [-1, 999] and kept[:2].tolist() == [0, 1] and math.isinf(logp[0]) and torch.equal(y[2], x[2])
    assert D.sample_rows(x, torch.tensor([0.5, 0.5, 0.5], device=DEV))[0][2] == token[2]


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_views_and_in_place(D, dtype):
    """Rows off every boundary, padded pitches, texts and masks inside larger buffers, results inside others, and over the logits."""
    R, V, L = 5, 1237, 40
    g = torch.Generator().manual_seed(12)
    big = (torch.randn(R, V + 20, generator=g) * 2).to(dtype).to(DEV)
    x = big[:, 3:3 + V]
    t = texts(R, L + 9, V, 13).to(DEV)[:, 4:4 + L]
    allowed = torch.rand(R, V, generator=g) < 0.7
    words = torch.zeros(R, 50, dtype=torch.int32, device=DEV)
    words[:, 2:2 + 39] = bits(allowed).to(DEV)
    bias = torch.randn(2 * V, generator=g).to(DEV)[::2]
    kw = dict(repetition=1.3, frequency=0.2, bias=bias, allowed=words[:, 2:2 + 39])
    want = D.adjust_rows(x.contiguous(), t.contiguous(), repetition=1.3, frequency=0.2, bias=bias.contiguous(), allowed=bits(allowed).to(DEV))
    check(want, *expected(x.cpu(), t.cpu(), repetition=1.3, frequency=0.2, bias=bias.cpu(), allowed=allowed), dtype)
    assert torch.equal(D.adjust_rows(x, t, **kw), want)
    out = torch.full((R, V + 11), 7.0, dtype=dtype, device=DEV)
    assert D.adjust_rows(x, t, out=out[:, 5:5 + V], **kw).data_ptr() == out[:, 5:].data_ptr()
    assert torch.equal(out[:, 5:5 + V], want) and (out[:, :5] == 7).all() and (out[:, 5 + V:] == 7).all()
    before = big.clone()
    D.adjust_rows(x, t, out=x, **kw)
    assert torch.equal(x, want) and torch.equal(big[:, :3], before[:, :3]) and torch.equal(big[:, 3 + V:], before[:, 3 + V:])
    three = before[:4, 3:3 + V].contiguous().view(2, 2, V)
    got = D.adjust_rows(three, t[:4].contiguous().view(2, 2, L), repetition=1.3, frequency=0.2, bias=bias, allowed=words[:4, 2:2 + 39])
    assert got.shape == (2, 2, V) and torch.equal(got.view(4, V), want[:4])
    one = D.adjust_rows(before[0, 3:3 + V], t[0], repetition=1.3, frequency=0.2, bias=bias, allowed=words[0, 2:2 + 39])
    assert one.shape == (V,) and torch.equal(one, want[0])
    assert D.adjust_rows(x[:0], t[:0]).shape == (0, V)


def test_the_same_bits_in_any_company(D):
    g = torch.Generator().manual_seed(14)
    x = torch.randn(300, 33000, generator=g).to(torch.bfloat16).to(DEV)
    t = texts(300, 500, 33000, 15).to(DEV)
    kw = dict(repetition=1.2, frequency=0.1, presence=0.3)
    whole = D.adjust_rows(x, t, **kw)
    for rows in (slice(0, 1), slice(7, 20), slice(100, 300)):
        assert torch.equal(D.adjust_rows(x[rows], t[rows], **kw), whole[rows])


# ---- the gradient

def expected_grad(g, x, tokens=None, token_rows=None, lengths=None, repetition=1.0, allowed=None, allowed_rows=None):
    R, V = g.shape
    by_x, kept = torch.empty(R, V, dtype=torch.float64), torch.empty(R, V, dtype=torch.float64)
    for r in range(R):
        _, seen = said(V, r, tokens, token_rows, lengths, 0)
        kept[r] = torch.where(mask_of(V, r, allowed, allowed_rows), g[r].double(), 0.0)
        rep = per_row(repetition, r)
        by_x[r] = torch.where(seen, torch.where(x[r] > 0, kept[r] / rep, kept[r] * rep), kept[r])
    return by_x, kept.sum(0), kept.abs().sum(0)


def check_grads(got, by_bias, want, dtype, bias_dtype, R):
    by_x, bias, size = want
    # one fp32 rounding and one to the type
    bound = (2.0 ** -24 + HALF_ULP[dtype]) * by_x.abs() * (1 + 2.0 ** -20) + STEP[dtype]
    assert ((got.double().cpu() - by_x).abs() <= bound).all()
    if by_bias is not None:                                   # R fp32 additions, each at most 2^-24 of the magnitudes' sum, and a rounding
        bound = (R + 1) * 2.0 ** -24 * size + HALF_ULP[bias_dtype] * bias.abs() * (1 + 2.0 ** -20) + STEP[bias_dtype]
        assert ((by_bias.double().cpu() - bias).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,L", [(1, 1, 1), (3, 33, 5), (70, 1001, 64), (130, 4099, 20), (33, 40000, 1200)])
def test_gradient(D, dtype, R, V, L):
    g = torch.Generator().manual_seed(R + V)
    x = (torch.randn(R, V, generator=g) * 2).to(dtype)
    x[:, ::5] = 0
    grad = torch.randn(R, V, generator=g).to(dtype)
    t = texts(3, L, V, 3)
    token_rows = torch.arange(R).mul(3).div(R, rounding_mode="floor").int()
    lengths = (torch.arange(R) % (L + 1)).int()
    allowed = torch.rand(2, V, generator=g) < 0.5
    allowed_rows = torch.randint(-1, 2, (R,), generator=g).int()
    rep = settings(R, 4)["repetition"]
    want = expected_grad(grad, x, t, token_rows, lengths, rep, allowed, allowed_rows)
    kw = dict(token_rows=token_rows.to(DEV), lengths=lengths.to(DEV), repetition=rep.to(DEV), allowed=bits(allowed).to(DEV), allowed_rows=allowed_rows.to(DEV))
    for bias_dtype in {torch.float32, dtype}:
        got, by_bias = D.adjust_grad(grad.to(DEV), x.to(DEV), t.to(DEV), want_bias=True, bias_dtype=bias_dtype, **kw)
        check_grads(got, by_bias, want, dtype, bias_dtype, R)
        assert by_bias.dtype == bias_dtype
        alone, none = D.adjust_grad(grad.to(DEV), x.to(DEV), t.to(DEV), **kw)
        assert none is None and torch.equal(alone, got)
        none, alone = D.adjust_grad(grad.to(DEV), want_logits=False, want_bias=True, bias_dtype=bias_dtype, allowed=kw["allowed"], allowed_rows=kw["allowed_rows"])
        assert none is None and torch.equal(alone, by_bias)


def test_masked_places_stop_nan_and_views_are_taken(D):
    R, V = 9, 777
    g = torch.Generator().manual_seed(5)
    big = torch.randn(R, V + 9, generator=g).to(torch.bfloat16)
    allowed = torch.rand(R, V, generator=g) < 0.5
    big[:, 2:2 + V] = torch.where(allowed, big[:, 2:2 + V], torch.tensor([math.nan, math.inf])[torch.randint(2, (R, V), generator=g)].to(torch.bfloat16))
    x = torch.randn(R, V, generator=g).to(torch.bfloat16)
    x[0, :50] = math.nan                                      # not above 0
    t = texts(1, 100, V, 6)
    grad = big.to(DEV)[:, 2:2 + V]
    want = expected_grad(grad.cpu(), x, t, repetition=1.5, allowed=allowed)
    got, by_bias = D.adjust_grad(grad, x.to(DEV), t.to(DEV), repetition=1.5, allowed=bits(allowed).to(DEV), want_bias=True)
    check_grads(got, by_bias, want, torch.bfloat16, torch.float32, R)
    over, _ = D.adjust_grad(grad, x.to(DEV), t.to(DEV), repetition=1.5, allowed=bits(allowed).to(DEV), out=grad)
    assert over.data_ptr() == grad.data_ptr() and torch.equal(over, got)


def test_autograd_is_the_formula_and_the_differences(D):
    """Weighed sums of the results, their gradients by logits and biases of each kind against differences: away from 0 the results are straight
    lines, so that a difference over a step h is exact but for the roundings of the two values."""
    R, V, L = 4, 40, 12
    g = torch.Generator().manual_seed(20)
    x = torch.randn(R, V, generator=g)
    x = torch.where(x.abs() < 0.1, 0.5, x)
    t = texts(R, L, V, 21)
    allowed = torch.rand(R, V, generator=g) < 0.7
    w = torch.randn(R, V, generator=g)
    kw = dict(repetition=torch.tensor([1.5, 0.75, 1.0, 2.0], device=DEV), frequency=0.25, presence=0.5, allowed=bits(allowed).to(DEV))
    for shape in ((V,), (1, V), (R, V)):
        b = torch.randn(shape, generator=g)
        xs, bs = x.to(DEV).requires_grad_(), b.to(DEV).requires_grad_()
        y = D.adjust_logits(xs, t.to(DEV), bias=bs, **kw)
        assert torch.equal(y.detach(), D.adjust_rows(x.to(DEV), t.to(DEV), bias=b.to(DEV), **kw))
        weights = torch.where(allowed, w, 0.0).to(DEV)
        torch.where(allowed.to(DEV), y * weights, 0.0).sum().backward()
        rep = kw["repetition"].cpu()
        by_x, _, _ = expected_grad(w, x, t, repetition=rep, allowed=allowed)
        by_b = torch.where(allowed, w, 0.0).double()
        assert torch.allclose(xs.grad.cpu().double(), by_x, rtol=2.0 ** -22, atol=0)
        want = by_b if shape == (R, V) else by_b.sum(0).view(shape)
        assert bs.grad.shape == shape and (bs.grad.cpu().double() - want).abs().max() <= R * 2.0 ** -23 * by_b.abs().sum(0).max()
        h = 2.0 ** -5
        for r, v in ((0, int(t[0].clamp(0, V - 1)[0])), (1, 7), (2, 3), (3, int(t[3].clamp(0, V - 1)[1]))):
            def line(dx, db):
                x2, b2 = x.clone(), b.clone()
                x2[r, v] += dx
                b2.view(-1, V)[r if shape == (R, V) else 0, v] += db
                y2 = D.adjust_rows(x2.to(DEV), t.to(DEV), bias=b2.to(DEV), **kw).cpu().double()
                return torch.where(allowed, y2 * w.double(), 0.0).sum()
            # every value is at most 32: off by at most 6 * 2^-24 * 32, times its weight (below 4), for up to R values, both ways
            slack = 2 * R * 6 * 2.0 ** -24 * 32 * 4 / (2 * h)
            assert abs((line(h, 0) - line(-h, 0)) / (2 * h) - by_x[r, v]) <= slack
            assert abs((line(0, h) - line(0, -h)) / (2 * h) - want.view(-1, V)[r if shape == (R, V) else 0, v]) <= slack


def test_a_gradient_is_differentiated_again(D):
    R, V = 3, 100
    g = torch.Generator().manual_seed(22)
    x, b = torch.randn(R, V, generator=g).to(DEV).requires_grad_(), torch.randn(V, generator=g).to(DEV).requires_grad_()
    t = texts(R, 30, V, 23, padded=False).to(DEV)
    allowed = torch.rand(1, V, generator=g) < 0.8
    w = torch.randn(R, V, generator=g).to(DEV).requires_grad_()
    kw = dict(repetition=1.5, presence=0.25, allowed=bits(allowed).to(DEV))
    y = D.adjust_logits(x, t, bias=b, **kw)
    gx, gb = torch.autograd.grad(y, (x, b), grad_outputs=w, create_graph=True)
    u, v = torch.randn(R, V, generator=g).to(DEV), torch.randn(V, generator=g).to(DEV)
    (gx * u).sum().add((gb * v).sum()).backward()
    factor, _, _ = expected_grad(torch.ones(R, V), x.detach().cpu(), t.cpu(), repetition=1.5, allowed=allowed)
    want = factor * u.cpu().double() + torch.where(allowed, v.cpu().double(), 0.0)
    size = (factor * u.cpu().double()).abs() + v.cpu().double().abs()
    assert ((w.grad.cpu().double() - want).abs() <= 3 * 2.0 ** -24 * size).all()


def test_expanded_and_transposed_gradients(D):
    x = torch.randn(6, 64, device=DEV).requires_grad_()
    b = torch.zeros(64, device=DEV).requires_grad_()
    D.adjust_logits(x, bias=b).sum().backward()
    assert (x.grad == 1).all() and (b.grad == 6).all()
    x.grad = None
    w = torch.randn(64, 6, device=DEV)
    (D.adjust_logits(x).t() * w).sum().backward()
    assert torch.equal(x.grad, w.t())


def test_written_sampled_and_taught(D):
    """The run of the operators together: an integer head, adjusted logits, sampling; then the same distribution's loss and its gradient back through
    the adjustment, added to the embedding's, clipped."""
    B, V, W, steps = 6, 500, 128, 5
    g = torch.Generator().manual_seed(30)
    table = (torch.randn(V, W, generator=g) * 0.3).to(torch.bfloat16).to(DEV)
    head = D.quantize_rows(table)
    bias = torch.zeros(V, device=DEV).requires_grad_()
    allowed = torch.rand(1, V, generator=g) < 0.5
    words = bits(allowed).to(DEV)
    text = torch.full((B, steps + 1), -1, dtype=torch.int64, device=DEV)
    text[:, 0] = torch.arange(B, device=DEV)
    states = []
    for i in range(steps):
        h = D.embed_rows(table, text[:, i], scale=1.0)
        states.append(h)
        y = D.adjust_rows(D.matmul_rows(D.quantize_rows(h), head), text, repetition=1.3, presence=0.5, prompt=1, bias=bias.detach(), allowed=words)
        u = torch.rand(B, generator=g).to(DEV)
        text[:, i + 1] = D.sample_rows(y, u, top_k=20)[0]
    assert allowed[0][text[:, 1:].cpu()].all()
    rows = torch.stack(states, 1).reshape(B * steps, W)
    tab = table.clone().requires_grad_()
    logits = rows @ tab.t()
    at = torch.arange(B * steps, device=DEV)
    y = D.adjust_logits(logits, text, token_rows=(at // steps).int(), lengths=(at % steps + 1).int(), prompt=1, repetition=1.3, presence=0.5, bias=bias,
                        allowed=words)
    val, idx = D.teacher_topk(torch.randn(B * steps, V, generator=g).to(torch.bfloat16).to(DEV), 16)
    loss, grad = D.div_topk_rest(0.5, y.detach(), val, idx, grad_scale=1.0 / (B * steps))
    assert loss.isfinite().all() and grad.isfinite().all() and (grad[:, ~allowed[0]] == 0).all()
    y.backward(grad)
    assert tab.grad.isfinite().all() and (bias.grad[~allowed[0].to(DEV)] == 0).all()
    exact = math.sqrt(sum(float(t.double().square().sum()) for t in (tab.grad, bias.grad)))
    norm = D.clip_grads([tab.grad, bias.grad], exact / 2)
    assert abs(norm.item() - exact) <= 2.0 ** -23 * exact
    after = math.sqrt(sum(float(t.double().square().sum()) for t in (tab.grad, bias.grad)))
    assert abs(after - exact / 2) <= 2.0 ** -8 * exact       # (each element of the table's gradient is rounded to bf16)


def test_captured_calls_replay(D):
    """Forward and gradients in a graph, replayed over new inputs with eager work between; two graphs do not share their workspaces."""
    R, V, L = 70, 3001, 50
    g = torch.Generator(device=DEV).manual_seed(31)
    x, grad = torch.randn(R, V, generator=g, device=DEV), torch.randn(R, V, generator=g, device=DEV)
    t = torch.randint(V, (R, L), generator=g, device=DEV)
    kw = dict(repetition=1.5)
    eager = lambda: (D.adjust_rows(x, t, frequency=0.5, **kw), *D.adjust_grad(grad, x, t, want_bias=True, **kw))  # noqa: E731
    eager()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = eager()
        graphs.append((graph, outs))
    for k in range(4):
        x.normal_(generator=g), grad.normal_(generator=g), t.random_(0, V, generator=g)
        want = [v.clone() for v in eager()]
        for graph, outs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_a_captured_training_step_replays(D):
    """`adjust_logits` and its backward pass in one graph, as a training loop captures them: warmed up on a side stream, no eager graph alive."""
    R, V, L = 40, 5003, 30
    g = torch.Generator(device=DEV).manual_seed(37)
    x, b = torch.randn(R, V, generator=g, device=DEV, requires_grad=True), torch.randn(V, generator=g, device=DEV, requires_grad=True)
    t, up = torch.randint(V, (R, L), generator=g, device=DEV), torch.randn(R, V, generator=g, device=DEV)

    def step():
        y = D.adjust_logits(x, t, repetition=1.3, presence=0.5, bias=b)
        return (y.detach(), *torch.autograd.grad(y, (x, b), up))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        with torch.no_grad():
            x.normal_(generator=g), b.normal_(generator=g), t.random_(0, V, generator=g), up.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(outs, step()))


def test_another_stream(D):
    x, t = torch.randn(20, 9000, device=DEV), torch.randint(9000, (20, 100), device=DEV)
    want = D.adjust_rows(x, t, repetition=1.2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = D.adjust_rows(x, t, repetition=1.2)
    s.synchronize()
    assert torch.equal(got, want)


def test_addresses_beyond_32_bits(D):
    """Logits of more than 2^31 elements, texts of more than 4 GiB."""
    R, V = 17000, 131072
    x = torch.zeros((R, V), dtype=torch.bfloat16, device=DEV)
    x[-1, -5:] = 4.0
    x[0, :5] = 4.0
    t = torch.full((80000, 8192), -1, dtype=torch.int64, device=DEV)
    t[79999, 8191], t[79999, 0], t[3, 7] = V - 2, V - 2, 2
    token_rows = torch.full((R,), -1, dtype=torch.int32, device=DEV)
    token_rows[-1], token_rows[0] = 79999, 3
    D.adjust_rows(x, t, token_rows=token_rows, repetition=2.0, frequency=0.25, out=x)
    assert x[-1, -6:].tolist() == [0, 4, 4, 4, 1.5, 4] and x[0, :6].tolist() == [4, 4, 1.75, 4, 4, 0]
    assert x.view(torch.int16).count_nonzero().item() == 10
    _, by_bias = D.adjust_grad(x, want_logits=False, want_bias=True)
    assert by_bias[-5:].tolist() == [4, 4, 4, 1.5, 4] and by_bias[:5].tolist() == [4, 4, 1.75, 4, 4] and by_bias.count_nonzero().item() == 10


def test_more_rows_than_a_launch_takes(D):
    n, V = 2 ** 24 + 77, 5
    g = torch.Generator(device=DEV).manual_seed(32)
    x = torch.randn((n, V), generator=g, device=DEV, dtype=torch.bfloat16)
    t = torch.randint(V, (n, 2), generator=g, device=DEV, dtype=torch.int32)
    allowed = torch.randint(1, 32, (n, 1), generator=g, device=DEV, dtype=torch.int32)
    got = D.adjust_rows(x, t, repetition=2.0, frequency=0.5, allowed=allowed)
    back, by_bias = D.adjust_grad(x, x, t, repetition=2.0, allowed=allowed, want_bias=True)
    for rows in (slice(0, 2 ** 18), slice(2 ** 24 - 2 ** 18, n)):
        assert torch.equal(got[rows], D.adjust_rows(x[rows], t[rows], repetition=2.0, frequency=0.5, allowed=allowed[rows]))
        assert torch.equal(back[rows], D.adjust_grad(x[rows], x[rows], t[rows], repetition=2.0, allowed=allowed[rows])[0])
    bit = (allowed >> torch.arange(V, device=DEV)) & 1
    kept = x.double() * bit
    assert ((by_bias.double() - kept.sum(0)).abs() <= 2.0 ** -24 * 300 * kept.abs().sum(0)).all()      # (runs of up to 257 rows)


def test_refusals(D):
    x, t = torch.randn(4, 100, device=DEV), torch.randint(100, (4, 9), device=DEV)
    words = torch.zeros(4, 4, dtype=torch.int32, device=DEV)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    with pytest.raises(ValueError):
        D.adjust_rows(x, t, repetition=0.0)
    with pytest.raises(ValueError):
        D.adjust_rows(x, t, repetition=math.nan)
    for call in (lambda: D.adjust_rows(x.double(), t), lambda: D.adjust_rows(x, t.float()), lambda: D.adjust_rows(x, t.cpu()), lambda: D.adjust_rows(x.cpu(), t),
                 lambda: D.adjust_rows(x, t[:3]), lambda: D.adjust_rows(x, token_rows=i32(4)), lambda: D.adjust_rows(x, t, token_rows=i32(3)),
                 lambda: D.adjust_rows(x, t, token_rows=i32(4).long()), lambda: D.adjust_rows(x, t, lengths=i32(5)), lambda: D.adjust_rows(x, t, prompt=i32(4).float()),
                 lambda: D.adjust_rows(x, t, frequency=torch.zeros(3, device=DEV)), lambda: D.adjust_rows(x, bias=torch.zeros(99, device=DEV)),
                 lambda: D.adjust_rows(x, bias=torch.zeros(100, device=DEV).half()), lambda: D.adjust_rows(x, bias=torch.zeros(3, 100, device=DEV)),
                 lambda: D.adjust_rows(x, allowed=words[:, :3]), lambda: D.adjust_rows(x, allowed=words.long()), lambda: D.adjust_rows(x, allowed=words[:2]),
                 lambda: D.adjust_rows(x, allowed_rows=i32(4)), lambda: D.adjust_rows(x, allowed=words, allowed_rows=i32(2)), lambda: D.adjust_rows(x.t(), t),
                 lambda: D.adjust_rows(x, out=torch.empty(4, 99, device=DEV)), lambda: D.adjust_rows(x, out=torch.empty(4, 100, device=DEV).half()),
                 lambda: D.adjust_rows(x[:, 1:], out=x[:, :-1]), lambda: D.adjust_rows(x[:1].expand(4, 100)), lambda: D.adjust_grad(x, None, t),
                 lambda: D.adjust_grad(x, x[:3], t), lambda: D.adjust_grad(x, x.half(), t), lambda: D.adjust_grad(x, want_bias=True, bias_dtype=torch.float16),
                 lambda: D.adjust_grad(x, x, t, out=torch.empty(4, 99, device=DEV)), lambda: D.adjust_grad(x, x.clone(), out=x[:, :50]),
                 lambda: D.adjust_grad(x.clone(), x, t, out=x), lambda: D.adjust_grad(x, want_logits=False, out=x)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("repetition", [2.0 ** -100, 2.0 ** -64, 1e-3, 3.0, 2.0 ** 64, 2.0 ** 101])
def test_quotients_are_rounded_once(D, repetition):
    """x / repetition of ordinary numbers is the fp32 quotient bit for bit, whatever the penalty's size."""
    g = torch.Generator().manual_seed(40)
    x = torch.randn(1, 5000, generator=g).abs() * (2.0 ** -20 if repetition < 1 else 2.0 ** 20)
    got = D.adjust_rows(x.to(DEV), torch.arange(5000, device=DEV).unsqueeze(0), repetition=torch.tensor([repetition], device=DEV))
    assert torch.equal(got.cpu(), x / torch.tensor(repetition))


def test_gradients_of_any_layout(D):
    """What autograd hands down may be transposed over the batch, expanded, or a part of wider rows."""
    g = torch.Generator().manual_seed(41)
    x = torch.randn(3, 4, 100, generator=g).to(DEV)
    t = texts(12, 20, 100, 42).to(DEV)
    w = torch.randn(3, 4, 100, generator=g).to(DEV)
    want = None
    for weigh in (lambda y: (y * w).sum(), lambda y: (y.transpose(0, 1) * w.transpose(0, 1).contiguous()).sum(),
                  lambda y: (y.permute(2, 0, 1) * w.permute(2, 0, 1).contiguous()).sum(),
                  lambda y: (torch.nn.functional.pad(y, (3, 5)) * torch.nn.functional.pad(w, (3, 5))).sum()):
        xs = x.clone().requires_grad_()
        b = torch.zeros(100, device=DEV).requires_grad_()
        weigh(D.adjust_logits(xs, t, bias=b, repetition=1.5)).backward()
        if want is None:
            want = xs.grad, b.grad
        assert torch.equal(xs.grad, want[0]) and torch.equal(b.grad, want[1])


def test_a_compiled_step(D):
    g = torch.Generator().manual_seed(43)
    x, b = torch.randn(6, 80, generator=g).to(DEV).requires_grad_(), torch.randn(80, generator=g).to(DEV).requires_grad_()
    t = texts(6, 15, 80, 44).to(DEV)
    w = torch.randn(6, 80, generator=g).to(DEV)

    def step(x, b, t, w):
        return (torch.softmax(D.adjust_logits(x, t, bias=b, repetition=1.25, presence=0.5), 1) * w).sum()

    want = torch.autograd.grad(step(x, b, t, w), (x, b))
    got = torch.autograd.grad(torch.compile(step, backend="aot_eager", fullgraph=True)(x, b, t, w), (x, b))
    assert torch.equal(got[0], want[0]) and torch.allclose(got[1], want[1], rtol=2.0 ** -20, atol=2.0 ** -24)


def test_very_wide_rows(D):
    """More columns than one launch joins; a text at both ends."""
    V = 540_000_000
    x = torch.zeros((1, V), dtype=torch.bfloat16, device=DEV)
    x[0, 0], x[0, V - 1], x[0, V // 2] = 2.0, 3.0, -1.0
    y = D.adjust_rows(x, torch.tensor([[0, V - 1, V - 1, V // 2, V, -1]], device=DEV), repetition=2.0, frequency=0.25)
    assert y[0, 0] == 0.75 and y[0, V - 1] == 1.0 and y[0, V // 2] == -2.25 and y.count_nonzero().item() == 3
    _, by_bias = D.adjust_grad(x, want_logits=False, want_bias=True)
    assert by_bias[0] == 2.0 and by_bias[V - 1] == 3.0 and by_bias[V // 2] == -1.0 and by_bias.count_nonzero().item() == 3


@pytest.mark.parametrize("dtype", DTYPES)
def test_sums_of_many_full_rows(D, dtype):
    """Rows enough, and as wide as the parts of the larger workgroups."""
    R, V = 2100, 32768 if dtype != torch.float32 else 16384
    g = torch.Generator(device=DEV).manual_seed(45)
    grad, x = torch.randn((R, V), generator=g, device=DEV).to(dtype), torch.randn((R, V), generator=g, device=DEV).to(dtype)
    t = torch.randint(V, (3, 700), generator=g, device=DEV)
    at = torch.arange(R, device=DEV)
    kw = dict(token_rows=(at // 700).int(), lengths=(at % 700).int(), repetition=1.5, allowed=torch.randint(-2 ** 31, 2 ** 31 - 1, (1, V // 32), generator=g, device=DEV, dtype=torch.int64).int())
    got, by_bias = D.adjust_grad(grad, x, t, want_bias=True, **kw)
    assert torch.equal(got, D.adjust_grad(grad, x, t, **kw)[0])
    bit = ((kw["allowed"].view(-1, 1) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).view(-1)
    kept = grad.double() * bit
    assert ((by_bias.double() - kept.sum(0)).abs() <= 2.0 ** -24 * 66 * kept.abs().sum(0)).all()      # (runs of 64 rows, one rounding)
    some = torch.tensor([0, 1, 699, 700, 1399, 2099], device=DEV)
    small, _ = D.adjust_grad(grad[some], x[some], t, token_rows=kw["token_rows"][some], lengths=kw["lengths"][some], repetition=1.5, allowed=kw["allowed"])
    assert torch.equal(got[some], small)


def test_the_example_writes_and_learns_under_penalties():
    """It runs with an integer head and penalties, no token twice in a text where a presence penalty forbids it, and its gradients through the
    adjustment are those of the same formula in torch operations."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "on_policy.py")
    spec = importlib.util.spec_from_file_location("on_policy_example_too", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    import llm_distillery_amd as D
    assert all(math.isfinite(v) for v in example.train(steps=3, penalties=dict(repetition=1.2, presence=0.5), integers=True))
    m = example.Model(200, 64, DEV, 3, 2.0)
    first = torch.arange(8, device=DEV)
    u = torch.rand(12, 8, generator=torch.Generator(device=DEV).manual_seed(46), device=DEV)
    written, _ = m.write(first, 12, u, penalties=dict(presence=1e9), integers=True)
    for f, row in zip(first.tolist(), written.tolist()):
        assert len({f, *row}) == 13
    tokens = torch.cat([first.unsqueeze(1), written[:, :-1]], 1)
    at = torch.arange(96, device=DEV, dtype=torch.int32)
    w = torch.randn(96, 200, generator=torch.Generator(device=DEV).manual_seed(47), device=DEV).bfloat16()
    logits = m.logits(m.states(tokens)).detach().requires_grad_()
    D.adjust_logits(logits, tokens, token_rows=at // 12, lengths=at % 12 + 1, repetition=1.5, presence=0.25).backward(w)
    seen = torch.zeros(96, 200, dtype=torch.bool, device=DEV)
    for r in range(96):
        seen[r, tokens[r // 12, : r % 12 + 1]] = True
    want = torch.where(seen, torch.where(logits > 0, w.double() / 1.5, w.double() * 1.5), w.double())
    # an fp32 rounding, and one to bf16, whose eight significant bits leave at most half a step, 2^-8 of the value
    bound = (HALF_ULP[torch.bfloat16] + 2.0 ** -24) * want.abs() * (1 + 2.0 ** -20) + STEP[torch.bfloat16]
    assert ((logits.grad.double() - want).abs() <= bound).all()


def test_empty_texts_and_rows(D):
    """Texts of no tokens, in any shape, and logits of no rows."""
    x = torch.randn(2, 3, 100, device=DEV)
    for t in (torch.empty((2, 3, 0), dtype=torch.int64, device=DEV), torch.empty((6, 0), dtype=torch.int32, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV)):
        assert torch.equal(D.adjust_rows(x, t, repetition=2.0, presence=1.0), x)
        assert torch.equal(D.adjust_grad(x, x, t, repetition=2.0)[0], x)
    none = torch.empty((0, 100), device=DEV)
    assert D.adjust_rows(none, torch.empty((0, 5), dtype=torch.int64, device=DEV), repetition=2.0).shape == (0, 100)
    rows, by_bias = D.adjust_grad(none, want_bias=True)
    assert rows.shape == (0, 100) and by_bias.count_nonzero().item() == 0 and by_bias.shape == (100,)



@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V", [(1, 5), (7, 33), (512, 9001), (2100, 32768), (4096, 16384), (9000, 40)])
def test_the_sum_of_rows_is_rounded_once(D, dtype, R, V):
    """The gradient by a shared bias: a sum in 64 bits, off by at most R - 1 roundings of 2^-53 of the magnitudes' sum (as the one here is), and one
    rounding to fp32, or that and one more to a type of 16 bits."""
    grad = torch.randn((R, V), generator=torch.Generator(device=DEV).manual_seed(R), device=DEV).to(dtype)
    want, size = grad.double().sum(0), grad.double().abs().sum(0)
    for bias_dtype in {torch.float32, dtype}:
        _, by_bias = D.adjust_grad(grad, want_logits=False, want_bias=True, bias_dtype=bias_dtype)
        half = 2.0 ** -24 + (HALF_ULP[bias_dtype] if bias_dtype != torch.float32 else 0.0)
        assert ((by_bias.double() - want).abs() <= half * want.abs() * (1 + 2.0 ** -7) + 2 * R * 2.0 ** -53 * size + STEP[bias_dtype]).all()
        assert torch.equal(by_bias, D.adjust_grad(grad, want_bias=True, bias_dtype=bias_dtype)[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R", [4, 8, 96, 4096])
def test_sums_on_the_way_may_leave_fp32(D, dtype, R):
    """Finite sums of values near the type's largest, the positive ones first: within a run of rows, and whole runs of them."""
    big = torch.finfo(dtype).max / 2
    grad = torch.zeros((R, 20000), dtype=dtype, device=DEV)
    grad[: R // 2, ::3], grad[R // 2:, ::3] = big, -big
    grad[::4, 1::3], grad[1::4, 1::3], grad[2::4, 1::3] = 1.5 * big, 1.5 * big, -3 * big / 2
    grad[3::4, 1::3] = -1.5 * big
    grad[0, 2::3], grad[R - 1, 2::3] = big, 0.5 * big
    want = grad.double().sum(0)
    _, by_bias = D.adjust_grad(grad, want_logits=False, want_bias=True)
    assert want.abs().max() == 1.5 * big and torch.equal(by_bias, want.float())


def test_autograd_sees_what_is_written_in_place(D):
    """A backward pass that needs values which a later call has overwritten raises, and none that does not need them."""
    g = torch.Generator(device=DEV).manual_seed(50)
    x = torch.randn(4, 100, generator=g, device=DEV).requires_grad_()
    t, w = torch.randint(100, (4, 30), generator=g, device=DEV), torch.randn(4, 100, generator=g, device=DEV).requires_grad_()
    kw = dict(repetition=1.5, presence=3.0)
    y = D.adjust_logits(x, t, **kw)                           # (whose gradient goes by the logits' signs)
    want, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    over = y.detach()
    assert D.adjust_rows(over, t, out=over, **kw) is over and y._version == 1
    assert torch.equal(torch.autograd.grad(y.sum(), x, retain_graph=True)[0], want)
    into = torch.empty_like(over)
    D.adjust_rows(x.detach(), t, out=into, **kw)
    assert into._version == 1 and x._version == 0
    D.adjust_rows(x.detach(), t, out=x.detach(), **kw)
    assert x._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    z = (w * x).sum()
    D.adjust_grad(w.detach(), x.detach(), t, repetition=1.5, out=w.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    with torch.inference_mode():                              # (a tensor without a version)
        into = torch.zeros(4, 100, device=DEV)
        D.adjust_rows(into, bias=torch.ones(100, device=DEV), out=into)
    assert (into == 1).all()


def test_a_result_that_would_need_a_gradient_is_refused(D):
    x = torch.randn(4, 100, device=DEV, requires_grad=True)
    y, bias = x * 1, torch.ones(100, device=DEV)
    before = y.detach().clone()
    for call in (lambda: D.adjust_rows(y, bias=bias, out=y), lambda: D.adjust_rows(before, bias=bias, out=x), lambda: D.adjust_grad(before, out=y)):
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call()
    assert torch.equal(y, before) and y._version == 0
    with torch.no_grad():
        assert D.adjust_rows(y, bias=bias, out=y) is y
    assert torch.equal(y, before + 1) and y._version == 1


def test_a_repetition_that_is_zero_in_fp32_is_refused(D):
    x, t = torch.zeros(2, 9, device=DEV), torch.zeros((2, 3), dtype=torch.int64, device=DEV)
    for repetition in (1e-46, 2.0 ** -150, 1e-300):
        for call in (lambda: D.adjust_rows(x, t, repetition=repetition), lambda: D.adjust_grad(x, x, t, repetition=repetition)):
            with pytest.raises(ValueError, match="positive"):
                call()
    assert torch.equal(D.adjust_rows(x, t, repetition=2.0 ** -149), x)      # (0 / 2^-149)


def test_rows_without_columns(D):
    """In any shape: nothing to adjust, gradients of no columns, rows of no codes."""
    x = torch.empty((2, 3, 0), device=DEV)
    assert D.adjust_rows(x, torch.zeros((6, 4), dtype=torch.int64, device=DEV), repetition=2.0).shape == (2, 3, 0)
    rows, by_bias = D.adjust_grad(x, want_bias=True)
    assert rows.shape == (2, 3, 0) and by_bias.shape == (0,)
    q = D.quantize_rows(x)
    assert q.codes.shape == (6, 0) and (q.scales == 2.0 ** -100).all()


def test_a_captured_backward_pass_into_the_leaves(D):
    """`.backward()` in a graph: the leaves have been in no graph of eager calls, their gradients are the capture's own."""
    R, V, L = 40, 5003, 30
    g = torch.Generator(device=DEV).manual_seed(51)
    leaves = lambda: (torch.zeros(R, V, device=DEV, requires_grad=True), torch.zeros(V, device=DEV, requires_grad=True))  # noqa: E731
    t, up = torch.zeros((R, L), dtype=torch.int64, device=DEV), torch.zeros(R, V, device=DEV)

    def step(x, b):
        D.adjust_logits(x, t, repetition=1.3, presence=0.5, bias=b).backward(up)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    x, b = leaves()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(x, b)
    for _ in range(3):
        with torch.no_grad():
            x.normal_(generator=g), b.normal_(generator=g), t.random_(0, V, generator=g), up.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        eager = [v.detach().clone().requires_grad_() for v in (x, b)]
        step(*eager)
        torch.cuda.synchronize()
        assert torch.equal(x.grad, eager[0].grad) and torch.equal(b.grad, eager[1].grad)
