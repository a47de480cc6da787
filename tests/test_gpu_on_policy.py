"""The example program: a step's operators together, and a loss that falls."""
import importlib.util
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("on_policy_example", os.path.join(ROOT, "examples", "on_policy.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_a_student_learns_from_what_it_writes(example):
    losses = example.train(steps=40)
    assert all(math.isfinite(v) for v in losses)
    first, last = sum(losses[:5]) / 5, sum(losses[-5:]) / 5
    assert last < 0.8 * first, f"{first} -> {last}"


def test_written_tokens_are_what_the_head_and_the_sampler_say(example):
    """One step by hand, with torch's own embedding, and the loss's gradient at the tied table as the sum of its two shares."""
    import llm_distillery_amd as D
    m = example.Model(300, 64, "cuda", 3, 2.0)
    first = torch.arange(20, device="cuda")
    u = torch.rand(1, 20, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    tokens, logp = m.write(first, 1, u, top_k=5)
    h = torch.tanh(torch.zeros(20, 64, dtype=torch.bfloat16, device="cuda") @ m.mix.detach() + (m.table.detach()[first].float() * m.scale).bfloat16())
    logits = D.matmul_blocks(D.quantize_blocks(h @ m.out.detach()), D.quantize_blocks(m.gain * m.table.detach(), rows=128))
    again = D.sample_rows(logits, u[0], top_k=5)
    assert torch.equal(tokens[:, 0], again[0]) and torch.equal(logp[:, 0], again[1])
    assert all(int(t) in torch.topk(row, 5).indices.tolist() for t, row in zip(tokens[:, 0], logits.float()))
    batch = torch.randint(300, (4, 6), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    grad = torch.randn(24, 300, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda").bfloat16()
    m.logits(m.states(batch)).backward(grad)
    both = m.table.grad.clone()
    m.table.grad = None
    x = (m.table.float()[batch] * m.scale).bfloat16()        # torch's lookup: the same values, its gradient summed by atomics
    s, got = torch.zeros_like(x[:, 0]), []
    for i in range(6):
        s = torch.tanh(s @ m.mix + x[:, i])
        got.append(s)
    m.logits(torch.stack(got, 1).reshape(-1, 64)).backward(grad)
    err = (both.float() - m.table.grad.float()).norm() / m.table.grad.float().norm()
    assert err.item() <= 2.0 ** -7                            # both shares and their sum are rounded to bf16
