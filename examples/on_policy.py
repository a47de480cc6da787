"""On-policy distillation of a toy student, the operators of a step together as a training program calls them.

    python examples/on_policy.py [--steps N]

A step: the student writes (its head in 8-bit floating point, sampling, embedding of the drawn tokens), the teacher scores what was
written (its log-probs reduced to the stored form by `teacher_topk`), the loss compares both over the stored entries and the rest of
the vocabulary, and the gradient goes back through the head to the tied embedding, whose two shares autograd adds up.
Teacher and student are small recurrent models of one vocabulary; needs an MI355X."""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import llm_distillery_amd as D  # noqa: E402


class Model(torch.nn.Module):
    """h <- tanh(h A + scale * table[token]); logits = gain * (h B) table^T."""

    def __init__(self, vocab, width, device, seed, gain):
        super().__init__()
        g = torch.Generator(device=device).manual_seed(seed)
        self.table = torch.nn.Parameter((torch.randn(vocab, width, generator=g, device=device) * 0.1).bfloat16())
        self.mix = torch.nn.Parameter((torch.randn(width, width, generator=g, device=device) * 0.5 / width ** 0.5).bfloat16())
        self.out = torch.nn.Parameter((torch.randn(width, width, generator=g, device=device) / width ** 0.5).bfloat16())
        self.scale, self.gain = width ** 0.5 * 0.5, gain

    def states(self, tokens):
        """The states behind every token of [batch, length], as [batch * length, width]."""
        x = D.embed(self.table, tokens, self.scale)
        h, got = torch.zeros_like(x[:, 0]), []
        for i in range(tokens.shape[1]):
            h = torch.tanh(h @ self.mix + x[:, i])
            got.append(h)
        return torch.stack(got, 1).reshape(-1, h.shape[1])

    def logits(self, states):
        return self.gain * (states @ self.out @ self.table.t())

    @torch.no_grad()
    def write(self, first, length, u, **settings):
        """`length` tokens behind `first` [batch], drawn with the random numbers u [length, batch]: (tokens [batch, length], their
        log-probabilities).  The head is quantised once; every step quantises its few states."""
        head = D.quantize_blocks(self.gain * self.table, rows=128)
        h, token, tokens, logps = torch.zeros((first.shape[0], self.table.shape[1]), dtype=self.table.dtype, device=first.device), first, [], []
        for i in range(length):
            h = torch.tanh(h @ self.mix + D.embed_rows(self.table, token, scale=self.scale))
            token, logp, _ = D.sample_rows(D.matmul_blocks(D.quantize_blocks(h @ self.out), head), u[i], **settings)
            tokens.append(token)
            logps.append(logp)
        return torch.stack(tokens, 1), torch.stack(logps, 1)


def train(steps=60, vocab=2048, width=256, batch=64, length=24, k=64, beta=0.5, lr=3e-3, device="cuda", report=None):
    """Trains a student on its own continuations; the mean loss per token of every step."""
    student, teacher = (Model(vocab, width, device, seed, 2.0) for seed in (0, 1))
    optimizer = torch.optim.Adam(student.parameters(), lr=lr)
    g = torch.Generator(device=device).manual_seed(2)
    losses = []
    for step in range(steps):
        first = torch.randint(vocab, (batch,), generator=g, device=device)
        u = torch.rand(length, batch, generator=g, device=device)
        written, _ = student.write(first, length, u, temperature=1.0, top_p=0.98, top_k=200)
        tokens = torch.cat([first.unsqueeze(1), written[:, :-1]], 1)
        with torch.no_grad():
            val, idx = D.teacher_topk(teacher.logits(teacher.states(tokens)), k)
        logits = student.logits(student.states(tokens))
        rows, grad = D.div_topk_rest(beta, logits.detach(), val, idx, grad_scale=1.0 / logits.shape[0])
        optimizer.zero_grad()
        logits.backward(grad)
        optimizer.step()
        losses.append(D.reduce_sum(rows, 1.0 / logits.shape[0]))
        if report and (step % 10 == 0 or step + 1 == steps):
            report(f"step {step}: loss per token {losses[-1].item():.4f}")
    return [v.item() for v in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    train(ap.parse_args().steps, report=lambda line: print(line, flush=True))
