"""GPU sampling against its definition in whole numbers, computed here row by row in numpy and Python integers."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F = np.float32
COEF = [F(float.fromhex(h)) for h in ("0x1.5bba14p-10", "0x1.3cea88p-7", "0x1.c6b752p-5", "0x1.ebf9bcp-3", "0x1.62e42ap-1", "0x1p0")]


@pytest.fixture(scope="module")
def D():
    import llm_distillery_amd as d
    d._lib.load()
    return d


def weights(x, T):
    """(order, whole weights in that order, t in that order) of the tokens of a row that have a weight."""
    x = np.where(np.isnan(x), F(-np.inf), x.astype(F))
    top = x.max()
    if top == -np.inf:
        return None
    with np.errstate(all="ignore"):
        rate = F(1.4426950408889634) / F(T) if T > 0 else F(np.inf)
        t = np.where(x == top, F(0), (x - top) * rate) if np.isinf(rate) or np.isinf(top) else (x - top) * rate
    t = np.where(t >= F(-64), t, F(-64)).astype(F)
    n = np.rint(t)
    f = t - n
    p = np.full_like(f, COEF[0])
    for c in COEF[1:]:
        p = (p * f).astype(F) + c
    w = np.floor(np.ldexp(p.astype(np.float64), n.astype(np.int64) + 31)).astype(np.int64)
    order = np.argsort(-x, kind="stable")
    order = order[w[order] > 0]
    return order, w[order], t[order]


def choose(x, u, T, k, top_p, min_p):
    got = weights(x, T)
    if got is None:
        return -1, 0
    order, w, _ = got
    k = k if T > 0 else 1
    end = min(k, len(w)) if k > 0 else len(w)
    upto = [0]
    for v in w.tolist():
        upto.append(upto[-1] + v)
    if top_p < 1:
        limit = max(1, upto[end] * int(max(0.0, float(F(top_p))) * 2 ** 24) >> 24)
        end = next(i for i in range(1, end + 1) if upto[i] >= limit)
    least = int(min(1.0, max(0.0, float(F(min_p)))) * 2 ** 31)
    end = next((i for i in range(end) if w[i] < least), end)
    want = upto[end] * min(2 ** 24 - 1, int(max(0.0, float(F(u))) * 2 ** 24)) >> 24
    lo, hi = 0, end                                           # the last i with upto[i] <= want
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (mid, hi) if upto[mid] <= want else (lo, mid)
    return int(order[lo]), end


def check(D, x, u, T, k, top_p, min_p, view=None):
    """x [R, V] on the CPU; settings per row (lists)."""
    R = x.shape[0]
    dev = view if view is not None else x.to(DEV)
    tokens, logp, kept = D.sample_rows(dev, torch.tensor(u, dtype=torch.float32, device=DEV), temperature=torch.tensor(T, dtype=torch.float32, device=DEV),
                                       top_k=torch.tensor(k, dtype=torch.int32, device=DEV), top_p=torch.tensor(top_p, dtype=torch.float32, device=DEV),
                                       min_p=torch.tensor(min_p, dtype=torch.float32, device=DEV))
    tokens, logp, kept = tokens.cpu(), logp.cpu(), kept.cpu()
    logits = x.float().numpy()
    for r in range(R):
        token, n = choose(logits[r], u[r], T[r], k[r], top_p[r], min_p[r])
        assert (int(tokens[r]), int(kept[r])) == (token, n), f"row {r}: T={T[r]} k={k[r]} p={top_p[r]} m={min_p[r]} u={u[r]}"
        z = np.where(np.isnan(logits[r]), -np.inf, logits[r].astype(np.float64))
        if token < 0:
            assert logp[r] == -math.inf
        elif T[r] <= 0 or np.isinf(z.max()):
            assert abs(float(logp[r]) + math.log((z == z.max()).sum())) <= 1e-6
        else:
            z = z / float(F(T[r]))
            want = z[token] - z.max() - math.log(np.exp(z - z.max()).sum())
            # t is off by three roundings of 2^-24 of itself, the powers by 2^-22, their sum in fp32 by 2^-18
            assert abs(float(logp[r]) - want) <= 2.0 ** -18 + 2.0 ** -21 * abs(z[token] - z.max())


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.05), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.01), (0.7, 400, 1.0, 0.0), (0.0, 0, 1.0, 0.0),
            (1.0, 1, 0.5, 0.5), (1.5, 3000, 0.99, 1e-6), (1.0, 0, 0.0, 0.0), (1.0, 0, 0.3, 1.0), (2.0, 7, 0.2, 0.0), (0.05, 0, 0.9, 0.2)]


def rows(R, V, seed, std=2.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * std
    at = torch.randint(V, (R, min(V, 40)), generator=g)
    x.scatter_(1, at, 3 * std + torch.randn(at.shape, generator=g))
    return x.to(dtype), torch.rand(R, generator=g).tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 9, 64, 1000, 4097, 32000, 50257])
def test_every_setting(D, V, dtype):
    x, u = rows(len(SETTINGS), V, V, dtype=dtype)
    check(D, x, u, *map(list, zip(*SETTINGS)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_wide_rows(D, dtype):
    x, u = rows(len(SETTINGS), 128256, 5, dtype=dtype)
    check(D, x, u, *map(list, zip(*SETTINGS)))


@pytest.mark.parametrize("V,dtype", [(20000, torch.float32), (20000, torch.bfloat16), (70001, torch.float16)])
def test_flat_rows_hold_more_than_a_list_in_a_bin(D, V, dtype):
    """Nearly equal logits: whole rows fall into a few bins, which are narrowed by the logits' order."""
    g = torch.Generator().manual_seed(V)
    x = (1.0 + torch.randn(len(SETTINGS), V, generator=g) * 2.0 ** -8).to(dtype)
    u = torch.rand(len(SETTINGS), generator=g).tolist()
    check(D, x, u, *map(list, zip(*SETTINGS)))
    many = [(1.0, V // 2, 1.0, 0.0), (1.0, V - 1, 0.7, 0.0), (1.0, 0, 0.5, 0.9), (1.0, V // 3, 0.999, 0.97), (2.0, 2049, 1.0, 0.0), (1.0, 0, 1.0, 0.99)]
    check(D, x[:6], u[:6], *map(list, zip(*many)))


@pytest.mark.parametrize("value", [0.0, -0.0, 3.5, -3.3895313892515355e38, 3.3895313892515355e38])
def test_equal_logits_go_by_their_index(D, value):
    V = 9001
    x = torch.full((len(SETTINGS), V), value, dtype=torch.bfloat16)
    if value == 0.0:
        x[:, ::3] = -0.0                                      # equal to 0
    u = [i / len(SETTINGS) for i in range(len(SETTINGS))]
    check(D, x, u, *map(list, zip(*SETTINGS)))


def test_random_numbers_at_the_ends(D):
    x, _ = rows(8, 3000, 2)
    u = [0.0, 1.0 - 2.0 ** -24, 2.0 ** -24, 0.5, 2.0 ** -30, 0.99999, 1.0, -1.0]
    check(D, x, u, [1.0] * 8, [0] * 8, [1.0] * 8, [0.0] * 8)
    check(D, x, u, [1.0] * 8, [5] * 8, [0.9] * 8, [0.0] * 8)


def test_masks_infinities_and_nan(D):
    x, u = rows(10, 2000, 3)
    x[0] = -math.inf                                          # nothing left
    x[1, 1:] = -math.inf                                      # one token
    x[2, ::2] = -math.inf
    x[3, 100] = math.inf
    x[4, [5, 50, 500]] = math.inf                             # share the mass
    x[5, ::7] = math.nan
    x[6] = math.nan                                           # nothing left
    x[7, 1000:] = torch.finfo(torch.float32).min
    x[8] = torch.finfo(torch.float32).min                     # a row of a mask's lowest value: all alike
    x[9, :1999] = -math.inf
    for T, k, p, m in [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.9, 0.05), (0.0, 0, 1.0, 0.0), (1e-42, 0, 1.0, 0.0), (1e30, 0, 0.5, 0.0), (math.inf, 0, 1.0, 0.0)]:
        if T == math.inf:                                     # every finite logit counts the same
            keep = [1, 2, 5, 7, 8, 9]
            got = D.sample_rows(x[keep].to(DEV), torch.tensor([u[i] for i in keep], device=DEV), temperature=T)
            for j, i in enumerate(keep):
                live = torch.isfinite(x[i]).nonzero()[:, 0]
                assert int(got[2][j]) == len(live) and int(got[0][j]) in set(live.tolist())
            continue
        check(D, x, u, [T] * 10, [k] * 10, [p] * 10, [m] * 10)


def test_views_shapes_and_plain_numbers(D):
    x, u = rows(6, 777, 8, dtype=torch.bfloat16)
    wide = torch.full((6, 800), 50.0, dtype=torch.bfloat16, device=DEV)
    wide[:, 5:782] = x.to(DEV)
    check(D, x, u, [0.9] * 6, [30] * 6, [0.95] * 6, [0.0] * 6, view=wide[:, 5:782])
    dev, ud = x.to(DEV), torch.tensor(u, device=DEV)
    one = D.sample_rows(dev, ud, temperature=0.9, top_k=30, top_p=0.95)
    box = D.sample_rows(dev.view(2, 3, 777), ud.view(2, 3), temperature=0.9, top_k=30, top_p=0.95)
    assert all(torch.equal(a, b.view(-1)) for a, b in zip(one, box)) and box[0].shape == (2, 3)
    single = D.sample_rows(dev[4], ud[4], temperature=0.9, top_k=30, top_p=0.95)
    assert all(torch.equal(a[4], b) for a, b in zip(one, single))
    assert D.sample_rows(dev[:0], ud[:0])[0].shape == (0,)


def test_the_token_does_not_depend_on_the_batch(D):
    x, u = rows(300, 32000, 11, dtype=torch.bfloat16)
    dev, ud = x.to(DEV), torch.tensor(u, device=DEV)
    whole = D.sample_rows(dev, ud, temperature=0.9, top_p=0.97)
    for n in (1, 3, 40):
        part = D.sample_rows(dev[7:7 + n], ud[7:7 + n], temperature=0.9, top_p=0.97)
        assert torch.equal(part[0], whole[0][7:7 + n]) and torch.equal(part[2], whole[2][7:7 + n])


def test_frequencies_follow_the_distribution(D):
    """20000 draws from one row of 12 tokens: each count within five standard deviations."""
    n = 20000
    x = torch.tensor([2.0, 1.0, 0.0, -1.0, 0.5, 3.0, -4.0, 1.5, 2.5, -math.inf, 0.0, 1.0])
    g = torch.Generator().manual_seed(4)
    tokens, logp, kept = D.sample_rows(x.expand(n, 12).contiguous().to(DEV), torch.rand(n, generator=g).to(DEV), temperature=1.3)
    p = torch.softmax(x.double() / 1.3, 0)
    count = torch.bincount(tokens.cpu(), minlength=12).double()
    assert ((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1e-9).all() and (kept == 11).all()


def test_refusals(D):
    x, u = torch.zeros(3, 10, device=DEV), torch.zeros(3, device=DEV)
    for bad in (dict(u=u.cpu()), dict(u=u.double()), dict(u=u[:2]), dict(logits=x.cpu()), dict(logits=x.double()), dict(logits=x.t().contiguous().t()),
                dict(temperature=torch.ones(2, device=DEV)), dict(top_k=torch.ones(3, device=DEV)), dict(top_p=torch.ones(3)), dict(logits=x[:, :0])):
        with pytest.raises(RuntimeError):
            a = {"logits": x, "u": u, **bad}
            D.sample_rows(a.pop("logits"), a.pop("u"), **a)
    with pytest.raises(ValueError):
        D.sample_rows(x, u, top_k=-1)
    lib, p = D._lib.load(), x.data_ptr()
    t = torch.zeros(3, dtype=torch.int64, device=DEV).data_ptr()
    assert lib.dl_sample_rows(p, 0, 9, 3, 10, p, 0, 0, 0, 0, 1.0, 0, 1.0, 0.0, t, 0, 0, 0) == -3
    assert lib.dl_sample_rows(p, 0, 10, 3, 10, 0, 0, 0, 0, 0, 1.0, 0, 1.0, 0.0, t, 0, 0, 0) == -1
    assert lib.dl_sample_rows(p + 1, 0, 10, 3, 10, p, 0, 0, 0, 0, 1.0, 0, 1.0, 0.0, t, 0, 0, 0) == -6
    assert lib.dl_sample_rows(p, 0, 5000000, 3, 5000000, p, 0, 0, 0, 0, 1.0, 0, 1.0, 0.0, t, 0, 0, 0) == -4
    assert lib.dl_sample_rows(p, 5, 10, 3, 10, p, 0, 0, 0, 0, 1.0, 0, 1.0, 0.0, t, 0, 0, 0) == -2


@pytest.mark.parametrize("R,V,dtype", [(12, 90001, torch.bfloat16), (12, 90001, torch.float32), (270, 20000, torch.float16)])
def test_cuts_and_tokens_far_down_flat_rows(D, R, V, dtype):
    """A cut behind many lists' worth of tokens, the token anywhere ahead of it: near the first, in a bin of its own, near the cut."""
    x, u = rows(R, V, V + 1, dtype=dtype)
    u = [(0.0, 1.0 - 2.0 ** -24, 0.999, u[r], u[r], u[r])[r % 6] for r in range(R)]
    T = [(1.2, 1.5, 1.6, 2.5)[r % 4] for r in range(R)]
    p = [(0.9, 0.98, 0.995)[r % 3] for r in range(R)]
    check(D, x, u, T, [0] * R, p, [0.0] * R)


@pytest.mark.parametrize("R", [4, 300])
@pytest.mark.parametrize("T,dtype,top,edge,behind", [(1.0, torch.float32, 0.0, -11.090355, -11.095), (1.4426950408889634, torch.bfloat16, 20.0, 4.0, 3.984375),
                                                     (1.4426950408889634, torch.float16, 31.0, 0.0, -0.015625), (1.4426950408889634, torch.float32, 31.0, 15.0, 14.99)])
def test_top_k_whose_last_token_is_at_the_edge_of_a_bin(D, R, T, dtype, top, edge, behind):
    """A few tokens at t = -16 or -31 exactly, thousands just behind them (t = -31: without a weight), the k-th among either."""
    V = 20000
    x = torch.full((R, V), -30.0)
    for r in range(R):
        at = torch.randperm(V, generator=torch.Generator().manual_seed(r))
        x[r, at[0]], x[r, at[1:11]], x[r, at[11:5011]] = top, edge, behind
    k = [(5, 11, 12, 4000)[r % 4] for r in range(R)]
    u = [(1.0 - 2.0 ** -24, 0.0, 0.99999, 0.9999999)[r // 4 % 4] for r in range(R)]
    check(D, x.to(dtype), u, [T] * R, k, [1.0] * R, [0.0] * R)
