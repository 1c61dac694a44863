"""Embedding, layer norm and sampling as they are used together: the example, its gradients, one step in a graph, and the rewired encoder."""
import copy
import os
import sys

import pytest
import torch

import sten_b200 as sten
from conftest import ROOT
from gpu_util import cuda

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(ROOT, "examples"))
import generate_sparse_model as example  # noqa: E402


@pytest.fixture(scope="module")
def run():
    return example.main(["--steps", "5", "--vocab", "1003", "--hidden", "64", "--tokens", "12"])


def test_the_example_writes_tokens(run):
    tokens, log_probs = run["tokens"], run["log_probs"]
    assert tokens.shape == log_probs.shape == (8, 12) and bool(((tokens >= 0) & (tokens < 1003)).all()) and bool((log_probs <= 0).all())


def test_replayed_steps_are_those_of_single_calls(run):
    """The graph's steps, one after the other, against calls outside of it."""
    model, window = run["sparse"], run["prompt"][:, -3:].clone()
    with torch.no_grad():
        for i in range(12):
            drawn = sten.sample_tokens(model(window)[:, -1], run["uniform"][:, i], temperature=0.8, top_k=50, top_p=0.95)
            assert torch.equal(drawn.tokens, run["tokens"][:, i]) and torch.equal(drawn.log_prob, run["log_probs"][:, i])
            window = torch.cat([window[:, 1:], drawn.tokens[:, None]], 1)


def test_gradients_of_the_example_against_its_definition(run):
    """The dense model's gradients against the same model written with torch's operators in 64 bits.

    The fp32 products of the model (sums of up to 256 terms, in any order, two layers and the head, forward and backward) are what limits this: some 10^3
    roundings of 2^-24 follow one another, 6e-5 of a gradient's norm if all pointed one way."""
    model = run["model"]
    tokens = example.sequences(1003, 16, 12, seed=3)
    tokens[0, 4:] = 0
    model.zero_grad()
    example.loss_of(model, tokens).backward()
    twin = copy.deepcopy(model).double()
    twin.zero_grad()
    h = torch.nn.functional.embedding(tokens, twin.token, padding_idx=0) * twin.scale
    y = h
    for b in twin.blocks:
        before = torch.nn.functional.pad(y, (0, 0, 1, 0))[:, :-1]
        h = h + b.down(torch.nn.functional.gelu(b.up(torch.cat([y, before], -1))))
        y = torch.nn.functional.layer_norm(h, h.shape[-1:], b.weight, b.bias)
    logits = twin.head(y)[:, :-1]
    torch.nn.functional.cross_entropy(logits.reshape(-1, 1003), tokens[:, 1:].reshape(-1)).backward()
    for (name, p), q in zip(model.named_parameters(), twin.parameters()):
        assert p.grad is not None and float((p.grad.double() - q.grad).norm()) <= 6e-5 * float(q.grad.norm()) + 1e-12, name
    assert not model.token.grad[0].any()


def test_sparse_weights_train_through_the_operators(run):
    sparse = run["sparse"]
    tokens = example.sequences(1003, 8, 10, seed=4)
    sparse.zero_grad()
    example.loss_of(sparse, tokens).backward()
    for name in ("token", "blocks.0.weight", "blocks.1.bias"):
        g = dict(sparse.named_parameters())[name].grad
        assert g is not None and bool(torch.isfinite(g).all()) and bool(g.any())


def test_layer_norms_of_rewired_modules():
    """fuse_linear_epilogues(layer_norms=True): the same numbers as with torch's norms but for roundings of fp16, and off again."""
    transformers = pytest.importorskip("transformers")
    cfg = transformers.BertConfig(hidden_size=128, num_hidden_layers=2, num_attention_heads=4, intermediate_size=512, vocab_size=1000, max_position_embeddings=128)
    torch.manual_seed(0)
    model = transformers.BertModel(cfg, add_pooling_layer=False).half().to(cuda()).eval()
    sb = sten.SparsityBuilder()
    for n, mod in model.named_modules():
        if isinstance(mod, torch.nn.Linear) and "encoder.layer" in n:
            sb.set_weight(name=n + ".weight", initial_sparsifier=sten.GroupedNMSparsifier(n=2, m=4, g=16), out_format=sten.GroupedNMTensor)
    sparse = sb.sparsify_model_inplace(model)
    ids = torch.randint(0, 1000, (4, 128), generator=torch.Generator().manual_seed(1)).to(cuda())

    def forward():
        with torch.no_grad():
            return sparse.encoder(sparse.embeddings(input_ids=ids), attention_mask=None).last_hidden_state

    assert sten.fuse_linear_epilogues(sparse) == 6
    torchs = forward()
    assert sten.fuse_linear_epilogues(sparse, layer_norms=True) == 0
    calls, real = [], sten.fusion.layer_norm
    sten.fusion.layer_norm = lambda *a, **k: calls.append(1) or real(*a, **k)
    try:
        ours = forward()
    finally:
        sten.fusion.layer_norm = real
    assert len(calls) == 4
    assert float((ours.double() - torchs.double()).norm() / torchs.double().norm()) <= 5e-3
    sten.fuse_linear_epilogues(sparse)
    assert torch.equal(forward(), torchs)
