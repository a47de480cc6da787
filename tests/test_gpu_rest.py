"""GPU parity of the top-K divergence with the rest as an outcome: loss against the definition in float64, gradient against
autograd of that definition, and against differences of the kernel's own loss."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
STEP = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
REST_MIN = 2.0 ** -14


@pytest.fixture(scope="module")
def D():
    import llm_distillery_amd as d
    d._lib.load()
    return d


def outcomes(z, lp, ids, rest_min):
    """(log P, log Q) over the listed ids and the rest, of one row in float64; z has a graph.  ids distinct, all counting."""
    total = torch.logsumexp(z, 0)
    others = torch.ones(z.shape[0], dtype=torch.bool)
    others[ids] = False
    lq = z[ids] - total
    p = lp.exp()
    if others.any() and torch.isfinite(z[others]).any():
        lq = torch.cat([lq, (torch.logsumexp(z[others], 0) - total).view(1)])
        p = torch.cat([p, (1 - p.sum()).clamp_min(rest_min).view(1)])
    return (p / p.sum()).log(), lq


def divergence(lp, lq, beta):
    p, q = lp.exp(), lq.exp()
    if beta == 0:
        return (p * (lp - lq)).sum()
    if beta == 1:
        return (q * (lq - lp)).sum()
    lm = torch.logaddexp(lp + math.log(beta), lq + math.log1p(-beta))
    return (beta * p * (lp - lm) + (1 - beta) * q * (lq - lm)).sum()


def entries(t_val, t_idx, n, V):
    """The counting entries of a stored row, repeated ids added up: (ids, log masses) in float64."""
    got = {}
    for v, i in zip(t_val[:n].double().tolist(), t_idx[:n].tolist()):
        if 0 <= i < V and v != -math.inf:
            got[i] = got.get(i, 0.0) + math.exp(v)
    ids = torch.tensor(list(got), dtype=torch.long)
    return ids, torch.tensor([math.log(v) for v in got.values()], dtype=torch.float64)


def check(D, logits, t_val, t_idx, beta, T=1.0, row_map=None, t_cnt=None, rest_min=REST_MIN, scale=0.5, **hooks):
    R, V = logits.shape
    dev = {k: (v.to(DEV) if v is not None else None) for k, v in (("row_map", row_map), ("t_cnt", t_cnt))}
    loss, grad = D.div_topk_rest(beta, logits.to(DEV), t_val.to(DEV), t_idx.to(DEV), T=T, rest_min=rest_min, grad_scale=scale, **dev, **hooks)
    alone, none = D.div_topk_rest(beta, logits.to(DEV), t_val.to(DEV), t_idx.to(DEV), T=T, rest_min=rest_min, want_grad=False, **dev, **hooks)
    assert none is None and torch.equal(alone, loss)
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    loss, grad = loss.cpu().double(), grad.cpu().double()
    c = scale / T
    for r in range(R):
        t = r if row_map is None else int(row_map[r])
        if t < 0 or t >= t_val.shape[0]:
            assert loss[r] == 0 and (grad[r] == 0).all()
            continue
        ids, lp = entries(t_val[t], t_idx[t], t_val.shape[1] if t_cnt is None else int(t_cnt[t]), V)
        z = (logits[r].double() / T).requires_grad_(True)
        P, Q = outcomes(z, lp, ids, rest_min)
        want = divergence(P, Q, beta)
        want.backward()
        g = z.grad * c
        with torch.no_grad():
            # a log-probability of the student comes from scaled logits and their log-sum in log2 units, each rounded to
            # 2^-24 of itself a few times; that error moves an outcome's share of the loss by (p + q) (1 + |log p/q|) times it
            live = z[torch.isfinite(z)]
            E = 2.0 ** -21 * (4 + (live.abs().max().item() * 1.4427 if live.numel() else 0))
            share = (P.exp() + Q.exp()) * (1 + (P - Q).abs())
            A = share.sum().item()
            assert abs(loss[r].item() - want.item()) <= E * A, f"row {r}: {loss[r].item()} against {want.item()}"
            q = torch.softmax(z, 0)
            bound = q * (2 * A + 1)
            bound[ids] += share[: len(ids)]
            if len(P) > len(ids):
                others = torch.ones(V, dtype=torch.bool)
                others[ids] = False
                w = torch.where(others, q, 0.0) / q[others].sum()
                bound += w * share[-1]
                stash = 0.0 if logits.dtype == torch.float32 else 2.0 ** -11      # powers of two-byte rows wait as fp16
                extra = stash * g.abs() * others + 2.0 ** -39 * c * (share[-1] + Q[-1].exp() * A) * others
            else:
                extra = 0.0
            bound = bound * E * c + extra + HALF_ULP[logits.dtype] * g.abs() * (1 + 2.0 ** -6) + STEP[logits.dtype]
            bad = (grad[r] - g).abs() > bound
            assert not bad.any(), f"row {r}: {int(bad.sum())} entries off, worst ratio {((grad[r] - g).abs() / bound).max().item():.2f}"
    return loss, grad


def case(R, V, K, dtype, seed, std=2.0, mass=0.9, val=torch.float16, idx=torch.int32):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(R, V, generator=g) * std).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(R)]) if R else torch.zeros((0, K), dtype=torch.long)
    lp = torch.log_softmax(torch.randn(R, K, generator=g) * 2, 1) + math.log(mass)
    if R and K:
        logits.scatter_(1, ids, (lp + math.log(V) + 3 + torch.randn(R, K, generator=g)).to(dtype))
    return logits, lp.to(val), ids.to(idx)


BETAS = [0.0, 0.1, 0.5, 0.9, 1.0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,V,K", [(1, 5, 2), (3, 64, 1), (5, 1000, 30), (4, 4099, 100), (3, 20001, 257), (2, 50257, 100), (2, 65543, 40)])
@pytest.mark.parametrize("beta", BETAS)
def test_loss_and_gradient(D, dtype, R, V, K, beta):
    check(D, *case(R, V, K, dtype, V + R), beta, T=1.5)


@pytest.mark.parametrize("V,dtype", [(128256, torch.bfloat16), (100003, torch.bfloat16), (151936, torch.float16), (70001, torch.float32), (300001, torch.bfloat16)])
@pytest.mark.parametrize("hooks", [{}, {"no_wait": True}])
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_rows_in_parts(D, V, dtype, hooks, beta):
    """Rows cut into column parts, waiting for their partners or finished by the second launch."""
    check(D, *case(9, V, 200, dtype, V), beta, **hooks)


def test_the_two_ways_through_parts_agree_bit_for_bit(D):
    a = [t.to(DEV) for t in case(40, 128256, 100, torch.bfloat16, 1)]
    one, two = D.div_topk_rest(0.5, *a), D.div_topk_rest(0.5, *a, no_wait=True)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


@pytest.mark.parametrize("beta", BETAS)
def test_masked_rows_counts_and_types(D, beta):
    logits, tv, ti = case(12, 3000, 50, torch.bfloat16, 3, val=torch.float32, idx=torch.int64)
    rm = torch.tensor([3, -1, 0, 11, 12, 99, 5, 5, -7, 1, 2, 4], dtype=torch.int32)
    cnt = torch.tensor([50, 0, 1, 49, 50, 7, 50, 50, 50, 50, 50, 60], dtype=torch.int32)
    check(D, logits, tv, ti, beta, row_map=rm, t_cnt=cnt.clamp_max(50))
    got = D.div_topk_rest(beta, logits.to(DEV), tv.to(DEV), ti.to(DEV), row_map=rm.to(DEV), t_cnt=cnt.to(DEV))      # 60 of 50: all
    want = D.div_topk_rest(beta, logits.to(DEV), tv.to(DEV), ti.to(DEV), row_map=rm.to(DEV), t_cnt=cnt.clamp_max(50).to(DEV))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("V", [600, 128256])
@pytest.mark.parametrize("beta", BETAS)
def test_entries_that_do_not_count_and_ids_that_repeat(D, V, beta):
    logits, tv, ti = case(4, V, 40, torch.float32, 4, mass=0.6, val=torch.float32)
    ti[0, :5] = torch.tensor([-1, V, V + 9, 2 ** 30, -2 ** 31], dtype=torch.int32)
    tv[1, 3:9] = -math.inf
    ti[2, 10:13] = ti[2, 0]
    ti[2, 20] = ti[2, 21]
    ti[3, :] = 7                                              # one outcome holds all of it
    check(D, logits, tv, ti, beta)


def test_teacher_that_stores_all_of_its_mass(D):
    """The listed masses reach 1 (or pass it, rounded): the rest has rest_min of the sum."""
    for mass in (1.0, 1.001, 0.99995):
        for beta in BETAS:
            check(D, *case(3, 900, 60, torch.float32, 5, mass=mass), beta, rest_min=2.0 ** -10)


@pytest.mark.parametrize("beta", BETAS)
def test_a_rest_far_below_the_listed_ids(D, beta):
    """1 - listed mass would be 0 in fp32: the rest's own sum is what counts."""
    logits, tv, ti = case(3, 700, 20, torch.float32, 6)
    others = torch.ones_like(logits, dtype=torch.bool).scatter_(1, ti.long(), False)
    check(D, torch.where(others, logits - 40.0, logits), tv, ti, beta)


@pytest.mark.parametrize("beta", BETAS)
def test_no_column_outside_the_list(D, beta):
    logits, tv, ti = case(4, 30, 30, torch.float32, 7)
    check(D, logits, tv, ti, beta)                            # every column listed
    logits, tv, ti = case(4, 500, 30, torch.bfloat16, 8)
    others = torch.ones_like(logits, dtype=torch.bool).scatter_(1, ti.long(), False)
    inf = check(D, torch.where(others, torch.tensor(-math.inf, dtype=logits.dtype), logits), tv, ti, beta)
    # masked with the type's lowest value instead: the same
    low = D.div_topk_rest(beta, torch.where(others, torch.tensor(torch.finfo(torch.bfloat16).min, dtype=logits.dtype), logits).to(DEV), tv.to(DEV),
                          ti.to(DEV), grad_scale=0.5)
    assert torch.equal(low[0].cpu().double(), inf[0]) and torch.equal(low[1].cpu().double(), inf[1])


@pytest.mark.parametrize("V", [500, 128256])
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.bfloat16).min, -1e30])
def test_masked_columns_among_the_rest(D, V, low):
    logits, tv, ti = case(3, V, 30, torch.bfloat16, 9)
    others = torch.ones_like(logits, dtype=torch.bool).scatter_(1, ti.long(), False)
    half = others.clone()
    half[:, V // 2:] = False
    masked = torch.where(half, torch.tensor(low, dtype=logits.dtype), logits)
    for beta in (0.0, 0.5, 1.0):
        loss, grad = check(D, torch.where(half, torch.tensor(-math.inf, dtype=logits.dtype), logits), tv, ti, beta)
        got = D.div_topk_rest(beta, masked.to(DEV), tv.to(DEV), ti.to(DEV), grad_scale=0.5)
        assert torch.equal(got[0].cpu().double(), loss) and torch.equal(got[1].cpu().double(), grad)


@pytest.mark.parametrize("V", [400, 128256])
def test_rows_that_mask_everything_or_have_nothing_to_compare(D, V):
    logits, tv, ti = case(6, V, 10, torch.bfloat16, 10)
    logits[0] = -math.inf
    logits[1] = torch.finfo(torch.bfloat16).min
    logits[1].scatter_(0, ti[1].long(), -math.inf)
    cnt = torch.full((6,), 10, dtype=torch.int32)
    cnt[2] = 0                                                # no entries: the rest alone, on both sides
    for beta in BETAS:
        loss, grad = D.div_topk_rest(beta, logits.to(DEV), tv.to(DEV), ti.to(DEV), t_cnt=cnt.to(DEV))
        assert (loss[:2] == 0).all() and (grad[:2] == 0).all()
        assert abs(loss[2].item()) <= 1e-5 and grad[2].abs().max().item() <= 1e-5
        assert torch.isfinite(loss[3:]).all() and torch.isfinite(grad[3:]).all() and (loss[3:] > 0).all()


def test_a_listed_id_the_student_rules_out(D):
    logits, tv, ti = case(2, 300, 10, torch.float32, 11)
    logits[0, ti[0, 3].item()] = -math.inf
    p = tv[0, 3].float().exp().item()
    loss, grad = D.div_topk_rest(0.0, logits.to(DEV), tv.to(DEV), ti.to(DEV))
    assert loss[0].item() == math.inf and math.isfinite(loss[1].item())
    assert abs(grad[0, ti[0, 3].item()].item() + p) <= 1e-5 and torch.isfinite(grad).all()
    for beta in (0.1, 0.5, 1.0):
        loss, grad = D.div_topk_rest(beta, logits.to(DEV), tv.to(DEV), ti.to(DEV))
        assert torch.isfinite(loss).all() and torch.isfinite(grad).all() and grad[0, ti[0, 3].item()] == 0


@pytest.mark.parametrize("V", [400, 128256])
def test_nan_and_infinity_stay_in_their_row(D, V):
    logits, tv, ti = case(5, V, 10, torch.bfloat16, 12)
    logits[1, 5] = math.nan
    logits[3, V - 2] = math.inf
    loss, grad = D.div_topk_rest(0.5, logits.to(DEV), tv.to(DEV), ti.to(DEV))
    assert torch.isnan(loss[[1, 3]]).all()
    assert torch.isfinite(loss[[0, 2, 4]]).all() and torch.isfinite(grad[[0, 2, 4]]).all()
    masked = torch.tensor([0, -1, 2, -1, 4], dtype=torch.int32, device=DEV)
    loss2, grad2 = D.div_topk_rest(0.5, logits.to(DEV), tv.to(DEV), ti.to(DEV), row_map=masked)
    assert (loss2[[1, 3]] == 0).all() and (grad2[[1, 3]] == 0).all() and torch.equal(loss2[[0, 2, 4]], loss[[0, 2, 4]])


def test_views_and_gradient_buffers(D):
    logits, tv, ti = case(5, 777, 20, torch.bfloat16, 13)
    want = D.div_topk_rest(0.5, logits.to(DEV), tv.to(DEV), ti.to(DEV))
    wide = torch.full((5, 800), math.nan, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:780] = logits.to(DEV)
    out = torch.full((5, 790), 9.0, dtype=torch.bfloat16, device=DEV)
    got = D.div_topk_rest(0.5, wide[:, 3:780], tv.to(DEV), ti.to(DEV), grad_out=out[:, 1:778])
    assert torch.equal(got[0], want[0]) and torch.equal(out[:, 1:778], want[1]) and (out[:, :1] == 9).all() and (out[:, 778:] == 9).all()
    three = D.div_topk_rest(0.5, logits.to(DEV).view(1, 5, 777), tv.to(DEV), ti.to(DEV))
    assert three[1].shape == (1, 5, 777) and torch.equal(three[1][0], want[1])
    none = D.div_topk_rest(0.5, logits.to(DEV)[:0], tv.to(DEV), ti.to(DEV))
    assert none[0].shape == (0,) and none[1].shape == (0, 777)
    no_entries = D.div_topk_rest(0.5, logits.to(DEV), tv.to(DEV)[:, :0], ti.to(DEV)[:, :0])
    assert no_entries[0].abs().max().item() <= 1e-5


def test_most_entries(D):
    check(D, *case(2, 9000, 2048, torch.bfloat16, 14), 0.5)


def test_gradient_against_differences(D):
    logits, tv, ti = case(6, 300, 20, torch.float32, 15, std=1.0)
    g = torch.Generator().manual_seed(16)
    direction = (torch.rand(6, 300, generator=g) * 2 - 1)
    h = 0.02
    for beta in BETAS:
        loss, grad = D.div_topk_rest(beta, logits.to(DEV), tv.to(DEV), ti.to(DEV))
        up, down = (D.div_topk_rest(beta, (logits + s * h * direction).to(DEV), tv.to(DEV), ti.to(DEV), want_grad=False)[0].cpu().double() for s in (1, -1))
        slope = (up - down) / (2 * h)
        want = (grad.cpu().double() * direction.double()).sum(1)
        # third derivative along a direction of at most 1 per logit: below 16 (1 + the largest |log p/q|, at most 12 here)
        assert ((slope - want).abs() <= h * h / 6 * 16 * 13 + 2e-5 / h).all()


def test_refusals(D):
    logits, tv, ti = (t.to(DEV) for t in case(3, 50, 4, torch.float32, 17))
    for beta in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError):
            D.div_topk_rest(beta, logits, tv, ti)
    for kw in (dict(rest_min=0.0), dict(rest_min=1.0), dict(T=0.0), dict(T=-1.0)):
        with pytest.raises(ValueError):
            D.div_topk_rest(0.5, logits, tv, ti, **kw)
    for a in ((logits.cpu(), tv, ti), (logits, tv.cpu(), ti), (logits, tv, ti.float()), (logits, tv[:2], ti[:2]), (logits, tv[:, :3], ti), (logits.double(), tv, ti)):
        with pytest.raises(RuntimeError):
            D.div_topk_rest(0.5, *a)
    with pytest.raises(RuntimeError):
        D.div_topk_rest(0.5, logits, tv, ti, grad_out=logits)
    with pytest.raises(RuntimeError):
        D.div_topk_rest(0.5, logits, torch.zeros(3, 2049, device=DEV), torch.zeros(3, 2049, dtype=torch.int32, device=DEV))
    lib = D._lib.load()
    big = torch.zeros((1, 128256), dtype=torch.bfloat16, device=DEV)
    assert lib.dl_div_topk_rest_workspace_bytes(1, 1, 128256) > 0
    assert lib.dl_div_topk_rest(0.5, big.data_ptr(), 1, 128256, 1, 128256, 0, tv.data_ptr(), 2, ti.data_ptr(), 0, 4, 3, 0, 1.0, 0.1, 1.0,
                                logits.data_ptr(), 0, 0, 0, 0, 0, 0) == -7
    assert lib.dl_div_topk_rest(0.5, big.data_ptr(), 1, 600000, 1, 600000, 0, tv.data_ptr(), 2, ti.data_ptr(), 0, 4, 3, 0, 1.0, 0.1, 1.0,
                                logits.data_ptr(), 0, 0, 0, 0, 0, 0) == -4
    assert lib.dl_div_topk_rest(0.5, 0, 1, 100, 1, 100, 0, tv.data_ptr(), 2, ti.data_ptr(), 0, 4, 3, 0, 1.0, 0.1, 1.0, logits.data_ptr(), 0, 0, 0, 0, 0, 0) == -1


@pytest.mark.parametrize("V", [400, 128256])
@pytest.mark.parametrize("T", [1.0, 2.0])
@pytest.mark.parametrize("beta", BETAS)
def test_an_entry_that_both_sides_mask_adds_nothing(D, V, T, beta):
    """A stored log-prob of fp16's lowest value is an entry without mass; where the student masks its column as well, it adds nothing, as
    an entry that does not count."""
    logits, tv, ti = case(3, V, 12, torch.bfloat16, 18)
    for low in (-math.inf, torch.finfo(torch.bfloat16).min, -1e30):
        x = logits.clone()
        for r in range(3):
            x[r, ti[r, 4 + r].item()] = low
        got, want = (D.div_topk_rest(beta, x.to(DEV), v.to(DEV), ti.to(DEV), T=T)
                     for v in (tv.scatter(1, torch.tensor([[4], [5], [6]]), value) for value in (torch.finfo(torch.float16).min, -math.inf)))
        assert torch.isfinite(want[0]).all() and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("V", [400, 128256])
@pytest.mark.parametrize("dtype,low", [(torch.bfloat16, torch.finfo(torch.bfloat16).min), (torch.bfloat16, -1e30), (torch.float32, -1e10),
                                       (torch.float32, torch.finfo(torch.float32).min)])
def test_rows_of_a_low_finite_mask_count_for_nothing(D, V, dtype, low):
    """Every logit masked with a low value that the scaling leaves finite: the listed ones too."""
    logits, tv, ti = case(4, V, 10, dtype, 19)
    logits[1], logits[3] = low, low
    for T in (1.0, 2.0):
        for beta in BETAS:
            loss, grad = D.div_topk_rest(beta, logits.to(DEV), tv.to(DEV), ti.to(DEV), T=T)
            assert (loss[[1, 3]] == 0).all() and (grad[[1, 3]] == 0).all()
            assert torch.isfinite(loss).all() and torch.isfinite(grad).all() and (loss[[0, 2]] > 0).all()


@pytest.mark.parametrize("V", [600, 70001])
@pytest.mark.parametrize("shift", [0.0, 2.0 ** 15, -2.0 ** 15])
@pytest.mark.parametrize("beta", BETAS)
def test_only_differences_of_logits_count(D, V, shift, beta):
    """fp32 logits far from 0: what a probability is off by goes with the logits' distances from the largest, not with the logits."""
    logits, tv, ti = case(3, V, 50, torch.float32, 20)
    logits = (logits * 256).round() / 256 + shift             # exact in fp32 with and without the shift
    for T in (1.0, 1.5):
        loss, grad = D.div_topk_rest(beta, logits.to(DEV), tv.to(DEV), ti.to(DEV), T=T)
        for r in range(3):
            ids, lp = entries(tv[r], ti[r], 50, V)
            z = (logits[r].double() / T).requires_grad_(True)
            P, Q = outcomes(z, lp, ids, REST_MIN)
            want = divergence(P, Q, beta)
            want.backward()
            g = z.grad / T
            with torch.no_grad():
                # log2 of a probability is x a - top, one multiply-add with a off by 2^-23 of itself, less the log2 of a sum of
                # powers, a few roundings of 2^-22: in all 2^-21 (4 + the largest distance in log2 units), whatever top is.  From
                # there as in check()
                E = 2.0 ** -21 * (4 + (z.max() - z.min()).item() * 1.4427)
                share = (P.exp() + Q.exp()) * (1 + (P - Q).abs())
                A = share.sum().item()
                q = torch.softmax(z, 0)
                others = torch.ones(V, dtype=torch.bool)
                others[ids] = False
                bound = q * (2 * A + 1) + torch.where(others, q, 0.0) / q[others].sum() * share[-1]
                bound[ids] += share[:-1]
                bound = bound * E / T + HALF_ULP[torch.float32] * g.abs() * (1 + 2.0 ** -6) + STEP[torch.float32]
                assert abs(loss[r].item() - want.item()) <= E * A
                assert ((grad[r].cpu().double() - g).abs() <= bound).all()
