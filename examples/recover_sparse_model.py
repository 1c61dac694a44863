"""A language model made sparse, and its quality recovered by distillation from the dense one.

A small model learns sequences (its loss is the mean log-probability of the next token), its feed-forward and head weights become
grouped n:m, which costs it, and the sparse student is trained on the top log-probabilities that were kept of the dense teacher.
The score is the same operator that the training used: log-probability of every next token, with the entropy beside it.

    python examples/recover_sparse_model.py [--steps 150] [--vocab 8000]
"""
import argparse
import copy
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import sten_b200 as sten  # noqa: E402


class Model(torch.nn.Module):
    """Next token from the two before it."""

    def __init__(self, vocab, hidden):
        super().__init__()
        self.token = torch.nn.Embedding(vocab, hidden)
        self.up = torch.nn.Linear(2 * hidden, 4 * hidden)
        self.down = torch.nn.Linear(4 * hidden, hidden)
        self.head = torch.nn.Linear(hidden, vocab)

    def forward(self, tokens):
        h = self.token(tokens)
        both = torch.cat([h, torch.nn.functional.pad(h, (0, 0, 1, 0))[:, :-1]], -1)
        return self.head(h + self.down(torch.nn.functional.gelu(self.up(both))))


def sequences(vocab, batch, length, seed):
    """Every token is a function of the two before it most of the time."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(0, vocab, (batch, length), device="cuda", generator=gen)
    noise = torch.rand(batch, length, device="cuda", generator=gen)
    for i in range(2, length):
        follows = (x[:, i - 1] * 31 + x[:, i - 2] % 7) % (vocab // 16)
        x[:, i] = torch.where(noise[:, i] < 0.9, follows, x[:, i])
    return x


def score(model, tokens):
    """(mean log-probability of the next token, mean entropy)"""
    with torch.no_grad():
        s = sten.token_log_probs(model(tokens)[:, :-1], tokens[:, 1:])
    return float(s.log_prob.mean()), float(s.entropy.mean())


def train_dense(model, vocab, steps, lr=3e-3):
    optimizer = torch.optim.Adam(model.parameters(), lr=lr)
    for step in range(steps):
        x = sequences(vocab, 16, 64, step)
        loss = -sten.token_log_probs(model(x)[:, :-1], x[:, 1:]).log_prob.mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()


def make_sparse(model, n, m, g):
    sb = sten.SparsityBuilder()
    for name in ("up.weight", "down.weight", "head.weight"):
        sb.set_weight(name, initial_sparsifier=sten.GroupedNMSparsifier(n, m, g), out_format=sten.GroupedNMTensor)
        sb.set_weight_grad(name, inline_sparsifier=sten.WeightLayoutSparsifier(), tmp_format=sten.GroupedNMTensor,
                           external_sparsifier=sten.KeepAll(), out_format=sten.GroupedNMTensor)
    return sb.get_sparse_model(model)


def descend(model, lr):
    """Gradient descent; a sparse weight keeps its layout, and its kept values take their part of the gradient."""
    with torch.no_grad():
        for p in model.parameters():
            if isinstance(p, sten.SparseTensorWrapper):
                p.wrapped_tensor.val.sub_(p.grad.wrapped_tensor.val, alpha=lr)
            else:
                p.sub_(p.grad, alpha=lr)
            p.grad = None


def distill(student, teacher, vocab, steps, kept, temperature=2.0, lr=0.1):
    for step in range(steps):
        x = sequences(vocab, 16, 64, 10_000 + step)
        with torch.no_grad():
            t = sten.token_log_probs(teacher(x), top=kept, temperature=temperature)
        loss = sten.distillation_loss(student(x), t.top_ids, t.top_log_prob, remainder=True, temperature=temperature)
        loss.backward()
        descend(student, lr)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--vocab", type=int, default=8000)
    ap.add_argument("--hidden", type=int, default=256)
    ap.add_argument("--steps", type=int, default=150)
    ap.add_argument("--kept", type=int, default=32)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    teacher = Model(a.vocab, a.hidden).cuda()
    held_out = sequences(a.vocab, 32, 64, 1 << 20)
    train_dense(teacher, a.vocab, a.steps)
    student = make_sparse(copy.deepcopy(teacher), 2, 4, 16)
    results = {"dense": score(teacher, held_out), "sparse": score(student, held_out)}
    distill(student, teacher, a.vocab, a.steps, a.kept)
    results["distilled"] = score(student, held_out)
    for name, (log_prob, entropy) in results.items():
        print(f"{name:10s} log-probability of the next token {log_prob:7.3f}, entropy {entropy:6.3f}")
    return results


if __name__ == "__main__":
    main()
