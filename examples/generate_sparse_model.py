"""A small language model of sparse products that is trained for some steps and then writes: the operators between the products together.

Tokens become scaled rows of the embedding matrix, every layer is a sparse feed-forward block with a residual and a layer norm, and
the next token is sampled from the logits.  One decode step (embedding, layers, head, sampling) is one CUDA graph, replayed for every token.
Training goes through the same operators: the matrix's gradient is that of sorted tokens, the norms' those of all that goes in.

    python examples/generate_sparse_model.py [--steps 60] [--vocab 4000] [--tokens 32] [--temperature 0.8] [--top-k 50] [--top-p 0.95]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import sten_b200 as sten  # noqa: E402


class Block(torch.nn.Module):
    def __init__(self, hidden):
        super().__init__()
        self.up = torch.nn.Linear(2 * hidden, 4 * hidden)
        self.down = torch.nn.Linear(4 * hidden, hidden)
        self.weight = torch.nn.Parameter(torch.ones(hidden))
        self.bias = torch.nn.Parameter(torch.zeros(hidden))

    def forward(self, y, h, before):
        """y: the last norm of the residual stream h; before: the same of the position before.  Returns both for the next block."""
        out = self.down(torch.nn.functional.gelu(self.up(torch.cat([y, before], -1))))
        return sten.layer_norm(out, self.weight, self.bias, residual=h)


class Model(torch.nn.Module):
    """Next token from the last ``1 + blocks`` ones."""

    def __init__(self, vocab, hidden, blocks=2):
        super().__init__()
        self.token = torch.nn.Parameter(torch.randn(vocab, hidden) / hidden ** 0.5)
        self.blocks = torch.nn.ModuleList(Block(hidden) for _ in range(blocks))
        self.head = torch.nn.Linear(hidden, vocab)
        self.scale = hidden ** 0.5

    def forward(self, tokens):
        h = sten.embedding(tokens, self.token, scale=self.scale, padding_idx=0)
        y = h
        for block in self.blocks:
            before = torch.nn.functional.pad(y, (0, 0, 1, 0))[:, :-1]
            y, h = block(y, h, before)
        return self.head(y)


def sequences(vocab, batch, length, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(1, vocab, (batch, length), device="cuda", generator=gen)
    noise = torch.rand(batch, length, device="cuda", generator=gen)
    for i in range(1, length):
        x[:, i] = torch.where(noise[:, i] < 0.9, (x[:, i - 1] * 31 + 7) % (vocab // 16) + 1, x[:, i])
    return x


def loss_of(model, tokens):
    return -sten.token_log_probs(model(tokens)[:, :-1], tokens[:, 1:]).log_prob.mean()


def make_sparse(model):
    sb = sten.SparsityBuilder()
    for name, mod in model.named_modules():
        if isinstance(mod, torch.nn.Linear):
            sb.set_weight(name + ".weight", initial_sparsifier=sten.GroupedNMSparsifier(2, 4, 4), out_format=sten.GroupedNMTensor)
    return sb.get_sparse_model(model)


def generate(model, prompt, steps, uniform, **settings):
    """Tokens [batch, steps] behind the prompt and their log-probabilities among those that the settings leave."""
    window = prompt[:, -(1 + len(model.blocks)):].clone()
    u = torch.empty(len(prompt), device=prompt.device)

    def step():
        drawn = sten.sample_tokens(model(window)[:, -1], u, **settings)
        window.copy_(torch.cat([window[:, 1:], drawn.tokens[:, None]], 1))
        return drawn

    with torch.no_grad():
        kept = window.clone()
        side = torch.cuda.Stream()  # a step outside of the graph makes the weights' copies
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            u.copy_(uniform[:, 0])
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            drawn = step()
        window.copy_(kept)
        tokens, log_probs = [], []
        for i in range(steps):
            u.copy_(uniform[:, i])
            graph.replay()
            tokens.append(drawn.tokens.clone())
            log_probs.append(drawn.log_prob.clone())
    return torch.stack(tokens, 1), torch.stack(log_probs, 1)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--vocab", type=int, default=4000)
    ap.add_argument("--hidden", type=int, default=256)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=50)
    ap.add_argument("--top-p", type=float, default=0.95)
    a = ap.parse_args(argv)
    sten.set_dispatch_failure("raise")
    torch.manual_seed(0)
    model = Model(a.vocab, a.hidden).cuda()
    opt = torch.optim.Adam(model.parameters(), lr=2e-3)
    losses = []
    for i in range(a.steps):
        loss = loss_of(model, sequences(a.vocab, 64, 32, seed=i))
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    print(f"dense model, {a.steps} steps: loss {losses[0]:.3f} -> {losses[-1]:.3f}")
    sparse = make_sparse(model).eval()
    prompt = sequences(a.vocab, 8, 8, seed=999)
    uniform = torch.rand(8, a.tokens, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    tokens, log_probs = generate(sparse, prompt, a.tokens, uniform, temperature=a.temperature, top_k=a.top_k, top_p=a.top_p)
    print("sampled:", tokens[0].tolist(), f"mean log-probability {float(log_probs.mean()):.3f}")
    return {"model": model, "sparse": sparse, "prompt": prompt, "uniform": uniform, "tokens": tokens, "log_probs": log_probs}


if __name__ == "__main__":
    main()
