"""A sparse language model between its sparse products: the operators from tokens to hidden states, between the layers and from
logits back to tokens, as measurable cases.

``sample``   one token a row of logits by temperature, top-k, top-p and min-p from a given uniform number, and its log-probability
``embed``    scaled rows of an embedding matrix, and with ``train`` the gradient of the matrix
``norm``     layer norm of a tensor or of its sum with a residual, and with ``train`` the gradients of all that goes in

``run`` computes a case in its plain form (elementary operations, in 32 bits or 64), or, where ``own`` is true, through the
package's entry points.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_INF = float("inf")


def _named(case, name):
    return case if name is None else {**case, "name": name}


def _sample(dtype, rows, vocab, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, masked=0, name=None):
    return _named({"op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
                   "mixed": mixed, "masked": masked}, name)


def _embed(dtype, tokens, vocab, width, *, scale=1.0, padding=False, train=True, name=None):
    return _named({"op": "embed", "dtype": dtype, "tokens": tokens, "vocab": vocab, "width": width, "scale": scale, "padding": padding, "train": train}, name)


def _norm(dtype, rows, width, *, residual=False, params="same", eps=1e-5, train=True, name=None):
    return _named({"op": "norm", "dtype": dtype, "rows": rows, "width": width, "residual": residual, "params": params, "eps": eps, "train": train}, name)


def listed():
    return [
        # the next token of one sequence on the encoder's vocabulary: the smallest call, all latency
        _sample("f16", 1, 30522, temperature=0.8, top_k=50, top_p=0.9, name="sample_one"),
        # a decode step of 64 requests, each with settings of its own (greedy ones among them), a few tokens banned
        _sample("bf16", 64, 131072, mixed=True, masked=11, name="sample_decode_batch"),
        # a large decode batch by nucleus alone: no top-k that would leave few tokens to look at
        _sample("bf16", 256, 131072, top_p=0.95, name="sample_nucleus_batch"),
        # rollouts for a policy-gradient step: the model's own distribution, nothing cut off
        _sample("bf16", 1024, 131072, name="sample_rollouts"),
        # fp32 logits, a ragged vocabulary of which a third is banned by a grammar, all filters at once
        _sample("f32", 97, 50021, temperature=1.3, top_k=200, top_p=0.97, min_p=0.01, masked=16673, name="sample_ragged_fp32"),
        # the tokens of a decode step looked up: latency
        _embed("bf16", 64, 131072, 4096, scale=64.0, train=False, name="embed_step"),
        # fine-tuning the encoder in fp32 (32 x 384 tokens), the ends of the sequences padded
        _embed("f32", 12288, 30522, 1024, padding=True, name="embed_train_encoder"),
        # a training step over a large vocabulary: the gradient of the matrix is nearly all there is to write
        _embed("bf16", 16384, 131072, 4096, scale=64.0, name="embed_train_large"),
        # a decode step of 16 sequences: latency
        _norm("f16", 16, 1024, residual=True, eps=1e-12, train=False, name="norm_step"),
        # a training batch of the encoder (32 x 384 tokens): residual and norm, parameters in fp32
        _norm("f16", 12288, 1024, residual=True, params="f32", eps=1e-12, name="norm_train_encoder"),
        # a wide model's training batch
        _norm("bf16", 16384, 8192, name="norm_train_large"),
        # fp32, sizes that are multiples of nothing
        _norm("f32", 3333, 1023, name="norm_ragged_fp32"),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(("f32", "f16", "bf16"))
    op = rng.choice(("sample", "sample", "embed", "norm"))
    if op == "sample":
        vocab = _log_uniform(rng, 500, 131072) | rng.choice((0, 1))
        rows = _log_uniform(rng, 1, min(4096, (1 << 27) // vocab))
        return _sample(dtype, rows, vocab, temperature=rng.choice((1.0, 0.7, 1.3, 0.2)), top_k=rng.choice((0, 0, 1, 5, 40, 300, vocab // 2)),
                       top_p=rng.choice((1.0, 1.0, 0.5, 0.9, 0.99)), min_p=rng.choice((0.0, 0.0, 0.02, 0.2)), mixed=rng.random() < 0.25,
                       masked=rng.choice((0, 0, 7, vocab // 3)))
    if op == "embed":
        width = _log_uniform(rng, 64, 8192) + rng.choice((0, 0, 1))
        vocab = _log_uniform(rng, 500, min(131072, (1 << 28) // width))
        return _embed(dtype, _log_uniform(rng, 1, min(32768, (1 << 26) // width)), vocab, width, scale=rng.choice((1.0, round(math.sqrt(width), 3))),
                      padding=rng.random() < 0.5, train=rng.random() < 0.7)
    width = _log_uniform(rng, 64, 16384) + rng.choice((0, 0, 1))
    return _norm(dtype, _log_uniform(rng, 1, min(32768, (1 << 26) // width)), width, residual=rng.random() < 0.5, params=rng.choice(("same", "f32")),
                 eps=rng.choice((1e-5, 1e-12)), train=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _prepare_sample(c, gen):
    rows, vocab, dtype = c["rows"], c["vocab"], _DTYPES[c["dtype"]]
    x = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // vocab)
    for a in range(0, rows, step):  # a scale of a few units, every other row with one or two tokens far ahead
        y = torch.randn(min(rows, a + step) - a, vocab, device="cuda", generator=gen).mul_(2.5)
        ahead = torch.randint(0, vocab, (len(y), 2), device="cuda", generator=gen)
        y.scatter_add_(1, ahead, torch.rand(len(y), 2, device="cuda", generator=gen) * 12 * (torch.arange(a, a + len(y), device="cuda")[:, None] % 2))
        if c["masked"]:
            y[:, vocab - c["masked"]:] = -_INF
        x[a:a + len(y)] = y
    state = {"case": c, "logits": x, "uniform": torch.rand(rows, device="cuda", generator=gen)}
    if c["mixed"]:
        def pick(values, like):
            return torch.tensor(values, dtype=like, device="cuda")[torch.randint(0, len(values), (rows,), device="cuda", generator=gen)]
        state["settings"] = {"temperature": pick((0.0, 0.6, 0.8, 1.0, 1.2), torch.float32), "top_k": pick((0, 0, 20, 50, 1000), torch.int64),
                             "top_p": pick((1.0, 0.8, 0.9, 0.95), torch.float32), "min_p": pick((0.0, 0.0, 0.05), torch.float32)}
    else:
        state["settings"] = {k: c[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    return state


def _prepare_embed(c, gen):
    tokens, vocab = c["tokens"], c["vocab"]
    # words' frequencies fall with their rank: ids are spread evenly over their logarithm
    ids = torch.exp(torch.rand(tokens, device="cuda", generator=gen, dtype=torch.float64) * math.log(vocab)).long().clamp_(0, vocab - 1)
    if c["padding"]:
        ids[torch.rand(tokens, device="cuda", generator=gen) < 0.2] = 0
    w = torch.empty(vocab, c["width"], dtype=_DTYPES[c["dtype"]], device="cuda").normal_(std=0.05, generator=gen)
    state = {"case": c, "ids": ids, "weight": w}
    if c["train"]:
        w.requires_grad_(True)
        state["grad"] = torch.randn(tokens, c["width"], device="cuda", generator=gen).to(w.dtype)
    return state


def _prepare_norm(c, gen):
    rows, width, dtype = c["rows"], c["width"], _DTYPES[c["dtype"]]
    kept = torch.float32 if c["params"] == "f32" else dtype

    def hidden(scale, shift=0.0):
        return (torch.randn(rows, width, device="cuda", generator=gen) * scale + shift).to(dtype)
    state = {"case": c, "x": hidden(1.5, 0.25), "weight": (1 + 0.1 * torch.randn(width, device="cuda", generator=gen)).to(kept),
             "bias": (0.1 * torch.randn(width, device="cuda", generator=gen)).to(kept)}
    state["x"][:, width // 3] += 20.0  # a feature that stands out in every row, as models have them
    if c["residual"]:
        state["residual"] = hidden(1.0)
    if c["train"]:
        state["grads"] = [hidden(1.0)] + ([hidden(1.0)] if c["residual"] else [])
        for k in ("x", "residual", "weight", "bias"):
            if k in state:
                state[k].requires_grad_(True)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"sample": _prepare_sample, "embed": _prepare_embed, "norm": _prepare_norm}[case["op"]](case, gen)


# ------------------------------------------------------------------------------------------------ the plain forms
def _column(v, rows):
    """A setting of every row, in 64 bits."""
    return v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full((rows, 1), float(v), dtype=torch.float64, device="cuda")


def _plain_sample(s):
    c, x = s["case"], s["logits"]
    rows, vocab = x.shape
    temperature, top_k, top_p, min_p = (_column(s["settings"][k], rows) for k in ("temperature", "top_k", "top_p", "min_p"))
    greedy = temperature == 0
    x64 = x.double()
    top = x64.amax(1, keepdim=True)
    z = (x64 - top) / torch.where(greedy, 1.0, temperature)
    weight = torch.exp(z)
    keep = z >= torch.log(min_p)
    if c["mixed"] or c["top_k"] or c["top_p"] < 1:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        w = weight.gather(1, order)
        place = torch.arange(vocab, device=x.device)[None]
        among = (top_k <= 0) | (place < top_k)
        w = torch.where(among, w, 0.0)
        before = torch.cumsum(w, 1) - w
        among &= (top_p >= 1) | (before < top_p * w.sum(1, keepdim=True)) | (place == 0)
        keep &= torch.zeros_like(keep).scatter_(1, order, among)
    kept = torch.where(keep, weight, 0.0)
    up_to = torch.cumsum(kept, 1)
    total = up_to[:, -1:]
    drawn = (up_to > s["uniform"].double()[:, None] * total).int().argmax(1, keepdim=True)
    first = (x64 == top).int().argmax(1, keepdim=True)
    tokens = torch.where(greedy, first, drawn)
    log_prob = torch.where(greedy, 0.0, z.gather(1, tokens) - torch.log(total))
    return {"tokens": tokens[:, 0], "log_prob": log_prob[:, 0].float()}


def _plain_embed(s):
    c, w, ids = s["case"], s["weight"].detach(), s["ids"]
    out = {"out": (w[ids].float() * c["scale"]).to(w.dtype)}
    if c["train"]:
        g = s["grad"].float() * c["scale"]
        if c["padding"]:
            g = torch.where((ids == 0)[:, None], 0.0, g)
        out["d_weight"] = torch.zeros(w.shape, device=w.device).index_add_(0, ids, g).to(w.dtype)
    return out


def _plain_norm(s):
    c, x = s["case"], s["x"].detach()
    h = x
    out = {}
    if c["residual"]:
        h = out["sum"] = (x.float() + s["residual"].detach().float()).to(x.dtype)
    weight, bias = s["weight"].detach().float(), s["bias"].detach().float()
    h = h.float()
    centred = h - h.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + c["eps"])
    normal = centred * rstd
    out["y"] = (normal * weight + bias).to(x.dtype)
    if c["train"]:
        g = s["grads"][0].float()
        gw = g * weight
        dx = rstd * (gw - gw.mean(1, keepdim=True) - normal * (gw * normal).mean(1, keepdim=True))
        if c["residual"]:
            dx = dx + s["grads"][1].float()
        out["d_x"] = dx.to(x.dtype)
        if c["residual"]:
            out["d_residual"] = out["d_x"]
        out["d_weight"] = (g * normal).sum(0).to(s["weight"].dtype)
        out["d_bias"] = g.sum(0).to(s["bias"].dtype)
    return out


# ------------------------------------------------------------------------------------------------ the framework's operators
def _own_sample(s):
    import sten_b200 as sten
    o = sten.sample_tokens(s["logits"], s["uniform"], **s["settings"])
    return {"tokens": o.tokens, "log_prob": o.log_prob}


def _own_embed(s):
    import sten_b200 as sten
    c = s["case"]
    y = sten.embedding(s["ids"], s["weight"], scale=c["scale"], padding_idx=0 if c["padding"] else None)
    out = {"out": y.detach()}
    if c["train"]:
        out["d_weight"] = torch.autograd.grad(y, s["weight"], s["grad"])[0]
    return out


def _own_norm(s):
    import sten_b200 as sten
    c = s["case"]
    o = sten.layer_norm(s["x"], s["weight"], s["bias"], eps=c["eps"], residual=s.get("residual"))
    y, outputs = (o[0], list(o)) if c["residual"] else (o, [o])
    out = {"sum": outputs[1].detach()} if c["residual"] else {}
    out["y"] = y.detach()
    if c["train"]:
        names = ["x"] + (["residual"] if c["residual"] else []) + ["weight", "bias"]
        out.update(zip(["d_" + k for k in names], torch.autograd.grad(outputs, [s[k] for k in names], s["grads"])))
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"sample": _own_sample, "embed": _own_embed, "norm": _own_norm}[op](state)
    with torch.no_grad():
        return {"sample": _plain_sample, "embed": _plain_embed, "norm": _plain_norm}[op](state)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_sample_row(x, u, temperature, top_k, top_p, min_p):
    """One row, token by token of the order of their probabilities."""
    if temperature == 0:
        return torch.nonzero(x == x.max())[0, 0], torch.zeros((), dtype=torch.float64, device=x.device)
    logp = torch.log_softmax(x.double() / temperature, 0)
    value, at = torch.sort(logp, descending=True, stable=True)
    if 0 < top_k < len(x):
        value, at = value[:top_k], at[:top_k]
    if top_p < 1:
        share = torch.softmax(value, 0)
        count = 1 + int((torch.cumsum(share, 0)[:-1] < top_p).sum())
        value, at = value[:count], at[:count]
    if min_p > 0:
        wanted = value - value[0] >= math.log(min_p)
        value, at = value[wanted], at[wanted]
    at, back = torch.sort(at)
    share = torch.softmax(value[back], 0)
    chosen = torch.searchsorted(torch.cumsum(share, 0), u, right=True).clamp(max=len(at) - 1)
    return at[chosen[0]], torch.log(share[chosen[0]])


def _exact_sample(c, s):
    x, rows = s["logits"], c["rows"]
    of_row = {k: v.tolist() if isinstance(v, torch.Tensor) else [v] * rows for k, v in s["settings"].items()}
    u = s["uniform"].double()
    found = [_exact_sample_row(x[r], u[r:r + 1], *(of_row[k][r] for k in ("temperature", "top_k", "top_p", "min_p"))) for r in range(rows)]
    return {"tokens": torch.stack([f[0] for f in found]), "log_prob": torch.stack([f[1] for f in found])}


def _exact_embed(c, s):
    w, ids = s["weight"].detach(), s["ids"]
    out = {"out": torch.nn.functional.embedding(ids, w).double() * c["scale"]}
    if c["train"]:
        ids_sorted, order = torch.sort(ids, stable=True)
        d = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        present, counts = torch.unique_consecutive(ids_sorted, return_counts=True)
        d[present] = torch.segment_reduce(s["grad"][order].double(), "sum", lengths=counts, axis=0) * c["scale"]
        if c["padding"]:
            d[0] = 0
        out["d_weight"] = d
    return out


def _exact_norm(c, s):
    names = ["x"] + (["residual"] if c["residual"] else []) + ["weight", "bias"]
    leaf = {k: s[k].detach().double().requires_grad_(c["train"]) for k in names}
    h, outputs = leaf["x"], []
    out = {}
    if c["residual"]:
        total = leaf["x"] + leaf["residual"]
        out["sum"] = total.detach()
        h = total + (total.detach().to(s["x"].dtype).double() - total.detach())  # the norm is that of the sum as it is returned
        outputs.append(total)
    y = torch.nn.functional.layer_norm(h, (c["width"],), leaf["weight"], leaf["bias"], c["eps"])
    out["y"] = y.detach()
    if c["train"]:
        d = torch.autograd.grad([y] + outputs, [leaf[k] for k in names], [g.double() for g in s["grads"]])
        out.update(zip(["d_" + k for k in names], d))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "embed": _exact_embed, "norm": _exact_norm}[case["op"]](case, s)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "sample":  # the logits once; per row the number, the settings, the token and its log-probability
        elements = c["rows"] * c["vocab"]
        return {"bytes": elements * size + c["rows"] * (16 + (20 if c["mixed"] else 0)), "flops": 4 * elements}
    if c["op"] == "embed":  # rows read once each time they are looked up, the output; the incoming gradient and the matrix's
        elements = c["tokens"] * c["width"]
        bytes_ = 8 * c["tokens"] + 2 * elements * size
        if c["train"]:
            bytes_ += elements * size + c["vocab"] * c["width"] * size
        return {"bytes": bytes_, "flops": elements * (3 if c["train"] else 1)}
    elements = c["rows"] * c["width"]
    kept = 4 if c["params"] == "f32" else size
    units = 2 + (2 if c["residual"] else 0)                        # x and y, residual and sum
    if c["train"]:
        units += 2 + (1 if c["residual"] else 0)                   # the gradients that come in, the one that goes out
    return {"bytes": elements * size * units + c["width"] * kept * (4 if c["train"] else 2), "flops": elements * (22 if c["train"] else 8)}
