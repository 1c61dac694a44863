"""Scoring and distilling a language model whose weights were made sparse: the operators over its vocabulary, as measurable cases.

``token``    log-probabilities of given tokens, entropy, log-sum-exp and the top alternatives of every row of logits, and with
             ``train`` their gradient
``distill``  divergence of a student from a teacher of whom only the top log-probabilities were kept, and with ``train`` the
             gradient of the student's logits

``rows`` x ``vocab`` are the logits.  ``run`` computes a case in its plain form (elementary operations in 32 bits), or, where
``own`` is true, through the package's entry points.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_INF = float("inf")
_IGNORE = -100


def _token(dtype, rows, vocab, *, top=0, targets=True, temperature=1.0, train=False, masked=0, ignored=0, shifted=0, name=None):
    c = {"op": "token", "dtype": dtype, "rows": rows, "vocab": vocab, "top": top, "targets": targets, "temperature": temperature,
         "train": train, "masked": masked, "ignored": ignored, "shifted": shifted}
    return c if name is None else {**c, "name": name}


def _distill(dtype, rows, vocab, kept, *, remainder=False, temperature=1.0, train=True, weighted=False, padded=0, reduction="mean", name=None):
    c = {"op": "distill", "dtype": dtype, "rows": rows, "vocab": vocab, "kept": kept, "remainder": remainder, "temperature": temperature,
         "train": train, "weighted": weighted, "padded": padded, "reduction": reduction}
    return c if name is None else {**c, "name": name}


def listed():
    return [
        # one decoded token, its probability and five alternatives on the encoder's vocabulary: the smallest call, all latency
        _token("f16", 1, 30522, top=5, name="token_one"),
        # a decode step of 64 requests over a large vocabulary, twenty alternatives each, a few tokens banned
        _token("bf16", 64, 131072, top=20, temperature=0.7, masked=11, name="token_decode_batch"),
        # scoring the encoder benchmark's batch (32 x 384 tokens): log-probabilities and entropy
        _token("f16", 12288, 30522, name="token_score_batch"),
        # next-token scores of eight fp32 sequences of 512: the logits but the last of each sequence, a strided view
        _token("f32", 8 * 511, 30522, shifted=511, name="token_score_shifted_fp32"),
        # keeping a teacher's 64 best tokens of 4096 positions for distillation
        _token("bf16", 4096, 131072, top=64, targets=False, temperature=2.0, name="token_teacher_top"),
        # a policy-gradient step with an entropy bonus: log-probabilities and entropy forward, both gradients back
        _token("bf16", 2048, 131072, train=True, name="token_policy_step"),
        # fp32 fine-tuning on a ragged vocabulary: padded columns, ignored positions, gradients of the alternatives too
        _token("f32", 777, 32003, top=4, train=True, masked=3, ignored=40, name="token_train_ragged_fp32"),
        # distilling a handful of positions: latency
        _distill("f16", 16, 30522, 8, name="distill_small"),
        # an ordinary training batch (8 x 512 tokens) on a middling vocabulary
        _distill("bf16", 4096, 32768, 32, temperature=2.0, name="distill_batch"),
        # the largest: 8192 positions, a large vocabulary, the teacher's remaining mass as a bucket of its own
        _distill("bf16", 8192, 131072, 64, remainder=True, name="distill_large"),
        # fp32, sizes that are multiples of nothing, rows of weight zero (padding), teacher rows of uneven length
        _distill("f32", 1023, 50021, 17, remainder=True, temperature=1.5, weighted=True, padded=5, name="distill_ragged_fp32"),
        # validation: the divergence of every position, no gradient
        _distill("bf16", 2000, 100003, 100, train=False, reduction="none", name="distill_evaluate"),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(("f32", "f16", "bf16"))
    vocab = _log_uniform(rng, 500, 131072) | rng.choice((0, 1))
    most = (1 << 29) // vocab // (2 if dtype == "f32" else 1)
    rows = _log_uniform(rng, 1, min(12288, most))
    temperature = rng.choice((1.0, 1.0, 0.7, 2.0, 1.3))
    if rng.random() < 0.5:
        train = rng.random() < 0.5
        return _token(dtype, rows, vocab, top=rng.choice((0, 0, 1, 3, 8, 20, 50, 128)), targets=train or rng.random() < 0.8, temperature=temperature, train=train,
                      masked=rng.choice((0, 0, 7, vocab // 3)), ignored=rng.choice((0, rows // 5)))
    return _distill(dtype, rows, vocab, _log_uniform(rng, 1, 128), remainder=rng.random() < 0.5, temperature=temperature, train=rng.random() < 0.7,
                    weighted=rng.random() < 0.4, padded=rng.choice((0, 0, 1)), reduction=rng.choice(("mean", "sum", "none")))


def _slabs(rows, vocab):
    """Ranges of rows whose 32- or 64-bit copies are small."""
    step = max(1, (1 << 26) // vocab)
    return [(r, min(rows, r + step)) for r in range(0, rows, step)]


def _student_logits(c, gen):
    """Rows as a model gives them: a scale of a few units, every other row with one or two tokens far ahead."""
    rows, vocab, dtype = c["rows"], c["vocab"], _DTYPES[c["dtype"]]
    x = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    for a, b in _slabs(rows, vocab):
        y = torch.randn(b - a, vocab, device="cuda", generator=gen).mul_(2.5)
        ahead = torch.randint(0, vocab, (b - a, 2), device="cuda", generator=gen)
        y.scatter_add_(1, ahead, torch.rand(b - a, 2, device="cuda", generator=gen) * 12 * (torch.arange(a, b, device="cuda")[:, None] % 2))
        if c.get("masked"):
            y[:, vocab - c["masked"]:] = -_INF
        x[a:b] = y
    return x


def _prepare_token(c, gen):
    rows, vocab = c["rows"], c["vocab"]
    x = _student_logits(c, gen)
    state = {"case": c}
    if c["targets"]:  # drawn from the model's own distribution, as sampled tokens are
        t = torch.empty(rows, dtype=torch.int64, device="cuda")
        for a, b in _slabs(rows, vocab):
            u = torch.rand(b - a, vocab, device="cuda", generator=gen).clamp_(min=1e-20)
            t[a:b] = (x[a:b].float() - u.log_().neg_().log_()).argmax(1)
        if c["ignored"]:
            t[torch.randperm(rows, device="cuda", generator=gen)[:c["ignored"]]] = _IGNORE
    if c["shifted"]:  # whole sequences, of which the scores of all positions but the last are wanted
        per = c["shifted"]
        full = torch.empty(rows // per, per + 1, vocab, dtype=x.dtype, device="cuda")
        full[:, :per] = x.view(rows // per, per, vocab)
        full[:, per] = full[:, 0]
        state["logits"] = full[:, :-1]
        tokens = torch.empty(rows // per, per + 1, dtype=torch.int64, device="cuda")
        tokens[:, 1:] = t.view(rows // per, per)
        tokens[:, 0] = 0
        state["targets"] = tokens[:, 1:]
    else:
        state["logits"], state["targets"] = x, t if c["targets"] else None
    if c["train"]:
        state["logits"].requires_grad_(True)
        state["grads"] = [torch.randn(rows, device="cuda", generator=gen) / rows for _ in range(2)]
        if c["top"]:
            state["grads"].append(torch.randn(rows, c["top"], device="cuda", generator=gen) / rows)
    return state


def _prepare_distill(c, gen):
    rows, vocab, kept = c["rows"], c["vocab"], c["kept"]
    x = _student_logits(c, gen)
    ids = torch.empty(rows, kept, dtype=torch.int64, device="cuda")
    log_probs = torch.empty(rows, kept, device="cuda")
    for a, b in _slabs(rows, vocab):  # a teacher that the student is near to
        z = (x[a:b].float() * 0.9 + torch.randn(b - a, vocab, device="cuda", generator=gen)) / c["temperature"]
        top, at = z.topk(kept, dim=1)
        ids[a:b], log_probs[a:b] = at, top - z.logsumexp(1, keepdim=True)
    if c["padded"]:  # teacher rows of uneven length end in tokens of -1
        length = torch.randint(max(1, kept - c["padded"]), kept + 1, (rows, 1), device="cuda", generator=gen)
        ids.masked_fill_(torch.arange(kept, device="cuda")[None] >= length, -1)
    weight = None
    if c["weighted"]:
        weight = torch.rand(rows, device="cuda", generator=gen) + 0.5
        weight[torch.rand(rows, device="cuda", generator=gen) < 0.2] = 0.0
    state = {"case": c, "logits": x, "ids": ids, "log_probs": log_probs, "weight": weight}
    if c["train"]:
        x.requires_grad_(True)
        if c["reduction"] == "none":
            state["grad"] = torch.rand(rows, device="cuda", generator=gen) / rows
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_token(case, gen) if case["op"] == "token" else _prepare_distill(case, gen)


# ------------------------------------------------------------------------------------------------ the plain forms
def _log_sum_exp(z):
    m = z.amax(1, keepdim=True)
    return m + torch.log(torch.exp(z - torch.where(m == -_INF, 0.0, m)).sum(1, keepdim=True))


def _plain_token(s):
    c, x = s["case"], s["logits"].detach()
    x = x.reshape(-1, x.shape[-1]).float()
    z = x if c["temperature"] == 1.0 else x / c["temperature"]
    lse = _log_sum_exp(z)
    empty = lse == -_INF  # a row that the mask leaves nothing of
    logp = torch.where(empty, -_INF, z - lse)
    p = torch.exp(logp)
    plogp = torch.where(p == 0, 0.0, p * logp)
    entropy = -plogp.sum(1, keepdim=True)
    out = {"entropy": entropy[:, 0], "lse": lse[:, 0]}
    if c["targets"]:
        targets = s["targets"].reshape(-1, 1)
        wanted = targets != _IGNORE
        at = torch.where(wanted, targets, 0)
        out["log_prob"] = torch.where(wanted, logp.gather(1, at), 0.0)[:, 0]
    if c["top"]:
        out["top_ids"] = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]].contiguous()
        out["top_log_prob"] = logp.gather(1, out["top_ids"])
    if c["train"]:
        g_log_prob, g_entropy = torch.where(wanted, s["grads"][0][:, None], 0.0), s["grads"][1][:, None]
        dz = -g_entropy * (plogp + p * entropy) - g_log_prob * p
        dz.scatter_add_(1, at, g_log_prob)
        if c["top"]:
            dz -= s["grads"][2].sum(1, keepdim=True) * p
            dz.scatter_add_(1, out["top_ids"], s["grads"][2])
        out["d_logits"] = torch.where(empty, 0.0, dz / c["temperature"]).to(s["logits"].dtype)
    return out


def _plain_distill(s):
    c, x, ids = s["case"], s["logits"].detach().float(), s["ids"]
    tau = c["temperature"]
    z = x if tau == 1.0 else x / tau
    lse = _log_sum_exp(z)
    valid = ids >= 0
    at = torch.where(valid, ids, 0)
    logq = torch.where(valid, s["log_probs"].float(), -_INF)
    if c["remainder"]:
        some = lse > -_INF
        rest = _log_sum_exp(torch.where(torch.zeros_like(z).scatter_add_(1, at, valid.float()) > 0, -_INF, z))
        q = torch.exp(logq)
        q_rest = torch.where(rest > -_INF, (1.0 - q.sum(1, keepdim=True)).clamp(min=0.0), 0.0)
    else:
        norm = _log_sum_exp(logq)
        some = (norm > -_INF) & (lse > -_INF)
        logq = torch.where(some, logq - norm, -_INF)
        q = torch.exp(logq)
    logp = z.gather(1, at) - lse
    loss = torch.where(q > 0, q * (logq - logp), 0.0).sum(1, keepdim=True)
    if c["remainder"]:
        loss = loss + torch.where(q_rest > 0, q_rest * (torch.log(q_rest) - (rest - lse)), 0.0)
    weight = torch.ones_like(loss) if s["weight"] is None else s["weight"][:, None]
    counts = some & (weight != 0)
    loss = torch.where(counts, tau * tau * weight * loss, 0.0)[:, 0]
    total = weight.sum() if c["reduction"] == "mean" else weight.new_ones(())
    out = {"loss": loss if c["reduction"] == "none" else torch.where(total != 0, loss.sum() / total, 0.0)}
    if c["train"]:
        p = torch.exp(z - lse)
        if c["remainder"]:
            mass = q.sum(1, keepdim=True) + q_rest
            others = torch.exp(z - rest) * (mass * torch.exp(rest - lse) - q_rest)
            there = torch.zeros_like(z).scatter_add_(1, at, valid.float()) > 0
            dz = torch.where(there, mass * p, others)
        else:
            dz = p
        dz = dz.scatter_add(1, at, -q)
        scale = tau * weight / torch.where(total != 0, total, 1.0)
        if c["reduction"] == "none":
            scale = scale * s["grad"][:, None]
        out["d_logits"] = torch.where(counts, scale * dz, 0.0).to(s["logits"].dtype)
    return out


# ------------------------------------------------------------------------------------------------ the framework's operators
def _own_token(s):
    import sten_b200 as sten
    c, x = s["case"], s["logits"]
    o = sten.token_log_probs(x, s["targets"], temperature=c["temperature"], top=c["top"])
    out = {"entropy": o.entropy.reshape(-1), "lse": o.lse.reshape(-1)}
    if c["targets"]:
        out["log_prob"] = o.log_prob.reshape(-1)
    if c["top"]:
        out["top_ids"], out["top_log_prob"] = o.top_ids, o.top_log_prob
    if c["train"]:
        outputs = [o.log_prob, o.entropy] + ([o.top_log_prob] if c["top"] else [])
        out["d_logits"] = torch.autograd.grad(outputs, x, s["grads"])[0]
        out = {k: v.detach() for k, v in out.items()}
    return out


def _own_distill(s):
    import sten_b200 as sten
    c = s["case"]
    loss = sten.distillation_loss(s["logits"], s["ids"], s["log_probs"], remainder=c["remainder"], weight=s["weight"], temperature=c["temperature"],
                                  reduction=c["reduction"])
    out = {"loss": loss.detach()}
    if c["train"]:
        out["d_logits"] = torch.autograd.grad(loss, s["logits"], s.get("grad"))[0]
    return out


def run(state):
    token = state["case"]["op"] == "token"
    if own:
        return _own_token(state) if token else _own_distill(state)
    with torch.no_grad():
        return _plain_token(state) if token else _plain_distill(state)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_token_rows(c, x, targets, grads):
    """The rows of ``x`` from torch's own log_softmax in 64 bits, the gradient by differentiating it."""
    x = x.double().requires_grad_(c["train"])
    logp = torch.log_softmax(x / c["temperature"], 1)
    out = {"lse": torch.logsumexp(x / c["temperature"], 1), "entropy": -torch.where(logp == -_INF, 0.0, logp.exp() * logp.clamp(min=-1e300)).sum(1)}
    if targets is not None:
        wanted = targets != _IGNORE
        out["log_prob"] = torch.where(wanted, logp[torch.arange(len(x), device=x.device), torch.where(wanted, targets, 0)], 0.0)
    if c["top"]:
        out["top_ids"] = None
        out["top_log_prob"] = logp.topk(c["top"], dim=1).values
    if c["train"]:
        total = (out["log_prob"] * grads[0].double()).sum() + (out["entropy"] * grads[1].double()).sum()
        if c["top"]:
            total = total + (out["top_log_prob"] * grads[2].double()).sum()
        out["d_logits"] = torch.autograd.grad(total, x)[0]
    return {k: v if v is None else v.detach() for k, v in out.items()}


def _exact_distill_rows(c, x, ids, log_probs, weight, grad):
    """Weighted divergence of every row, and the gradient of its sum with ``grad`` by differentiating it."""
    x = x.double().requires_grad_(c["train"])
    z = x / c["temperature"]
    valid = ids >= 0
    at = ids.clamp(min=0)
    logq = log_probs.double().masked_fill(~valid, -_INF)
    logp = torch.log_softmax(z, 1).gather(1, at)
    if c["remainder"]:
        hidden = torch.zeros(z.shape, dtype=torch.int32, device=z.device).scatter_add_(1, at, valid.int()) > 0
        log_rest = torch.logsumexp(z.masked_fill(hidden, -_INF), 1) - torch.logsumexp(z, 1)
        q_rest = (1 - logq.exp().sum(1)).clamp(min=0)
        tail = torch.special.xlogy(q_rest, q_rest) - q_rest * log_rest
    else:
        logq = torch.log_softmax(logq, 1)
        tail = 0.0
    terms = logq.exp() * (logq.masked_fill(~valid, 0.0) - logp.masked_fill(~valid, 0.0))
    loss = c["temperature"] ** 2 * weight * (terms.sum(1) + tail)
    d = torch.autograd.grad((loss * grad).sum(), x)[0] if c["train"] else None
    return loss.detach(), d


def exact(case, seed):
    c, s = case, prepare(case, seed)
    x = s["logits"].detach()
    x = x.reshape(-1, x.shape[-1])
    rows = c["rows"]
    if c["op"] == "token":
        targets = None if s["targets"] is None else s["targets"].reshape(-1)
        parts = [_exact_token_rows(c, x[a:b], None if targets is None else targets[a:b], [g[a:b] for g in s.get("grads", [])])
                 for a, b in _slabs(rows, c["vocab"])]
        return {k: None if parts[0][k] is None else torch.cat([q[k] for q in parts]) for k in parts[0]}
    weight = (torch.ones(rows, device="cuda") if s["weight"] is None else s["weight"]).double()
    total = float(weight.sum()) if c["reduction"] == "mean" else 1.0
    grad = s["grad"].double() if "grad" in s else torch.full((rows,), 1.0 / total if total else 0.0, dtype=torch.float64, device="cuda")
    parts = [_exact_distill_rows(c, x[a:b], s["ids"][a:b], s["log_probs"][a:b], weight[a:b], grad[a:b]) for a, b in _slabs(rows, c["vocab"])]
    loss = torch.cat([q[0] for q in parts])
    out = {"loss": loss if c["reduction"] == "none" else loss.sum() / total if total else torch.zeros((), dtype=torch.float64)}
    if c["train"]:
        out["d_logits"] = torch.cat([q[1] for q in parts])
    return out


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    elements, size = c["rows"] * c["vocab"], 4 if c["dtype"] == "f32" else 2
    # the logits once, and with a gradient that once; per row and kept token what is small beside them
    small = 12 * c["top"] + 8 * c["targets"] + 12 if c["op"] == "token" else 12 * c["kept"] + 4 * c["weighted"] + 4
    moved = elements * size * (2 if c["train"] else 1) + c["rows"] * (small + (8 + 4 * c.get("top", 0) if c["train"] and c["op"] == "token" else 0))
    # per element a difference, an exponential and an addition (the entropy: a product and an addition more); backward the probability and its scaling
    flops = elements * ((5 if c["op"] == "token" else 3) + (4 if c["train"] else 0))
    return {"bytes": moved, "flops": flops}
