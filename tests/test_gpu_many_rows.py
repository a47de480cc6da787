"""Calls whose rows or tokens are more than the threads of one launch (2^32) take: every row is there, up to the last."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def D():
    import llm_distillery_amd as d
    d._lib.load()
    return d


def test_sampled_rows(D):
    n = 2 ** 23 + 77
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((n, 3), generator=g, device=DEV, dtype=torch.bfloat16)
    u = torch.rand(n, generator=g, device=DEV)
    T = torch.rand(n, generator=g, device=DEV)
    k = torch.randint(3, (n,), generator=g, device=DEV, dtype=torch.int32)
    p = 0.5 + torch.rand(n, generator=g, device=DEV)
    m = 0.1 * torch.rand(n, generator=g, device=DEV)
    got = D.sample_rows(x, u, temperature=T, top_k=k, top_p=p, min_p=m)
    for rows in (slice(0, 2 ** 20), slice(2 ** 23 - 2 ** 20, n)):
        some = D.sample_rows(x[rows], u[rows], temperature=T[rows], top_k=k[rows], top_p=p[rows], min_p=m[rows])
        assert all(torch.equal(a[rows], b) for a, b in zip(got, some))


def test_lookup(D):
    n = 2 ** 26 + 77
    tokens = torch.arange(n, dtype=torch.int32, device=DEV) % 1000 - 1          # (-1: a row of zeros)
    table = torch.randn((999, 1), device=DEV)
    got = D.embed_rows(table, tokens)
    want = torch.cat([torch.zeros((1, 1), device=DEV), table])
    for part in range(0, n, 2 ** 24):
        at = slice(part, min(n, part + 2 ** 24))
        assert torch.equal(got[at], want[(tokens[at] + 1).long()])


def test_embedding_gradient(D):
    """More than 2^29 tokens (their tiles join in more workgroups of 256 than one launch takes): every row's sum is a whole number
    that fp32 holds."""
    n, vocab = 2 ** 29 + 200, 65536
    tokens = torch.arange(n, dtype=torch.int32, device=DEV) % vocab
    got = D.embed_grad(torch.ones((n, 1), dtype=torch.bfloat16, device=DEV), tokens, vocab, dtype=torch.float32)
    want = torch.full((vocab, 1), float(n // vocab), device=DEV)
    want[: n % vocab] += 1
    assert torch.equal(got, want)


@pytest.mark.parametrize("mapped", [False, True])
def test_divergence_with_the_rest(D, mapped):
    n = 2 ** 24 + 77
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn((n, 5), generator=g, device=DEV, dtype=torch.bfloat16)
    t = 1000 if mapped else n - 3                             # (without a map the last three rows have no teacher)
    val = -0.5 - torch.rand((t, 1), generator=g, device=DEV)
    idx = torch.randint(5, (t, 1), generator=g, device=DEV, dtype=torch.int32)
    cnt = torch.randint(2, (t,), generator=g, device=DEV, dtype=torch.int32)
    row_map = (torch.arange(n, device=DEV) % 1001 - 1).int() if mapped else (torch.arange(n, device=DEV)).int()
    loss, grad = D.div_topk_rest(0.5, x, val, idx, t_cnt=cnt, row_map=row_map)
    for rows in (slice(0, 2 ** 20), slice(2 ** 24 - 2 ** 20, n)):
        some = D.div_topk_rest(0.5, x[rows], val, idx, t_cnt=cnt, row_map=row_map[rows])
        assert torch.equal(loss[rows], some[0]) and torch.equal(grad[rows], some[1])
    if not mapped:
        more = torch.cat([val, val[:3]]), torch.cat([idx, idx[:3]])
        cnt = torch.cat([cnt, torch.zeros(3, dtype=torch.int32, device=DEV)])
        loss2, grad2 = D.div_topk_rest(0.5, x, *more, t_cnt=cnt)
        assert torch.equal(loss2[:-3], loss[:-3]) and torch.equal(grad2[:-3], grad[:-3])
        assert (loss[-3:] == 0).all() and (grad[-3:] == 0).all()


def test_more_columns_than_a_launch_takes_are_refused(D):
    lib, p = D._lib.load(), torch.zeros(4, device=DEV).data_ptr()
    cols = 2 ** 31
    for rows in (1, 128):
        assert lib.dl_quantize_blocks(p, 1, cols, 1, cols, rows, p, cols, p, 2 ** 24, 1, 0) == -4
