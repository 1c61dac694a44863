"""fuse_linear_epilogues(layer_norms=True) replaces a norm only where the call does what the module would have done."""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu


class Output(torch.nn.Module):
    def __init__(self, hidden=64):
        super().__init__()
        self.dense, self.dropout, self.LayerNorm = torch.nn.Linear(2 * hidden, hidden), torch.nn.Dropout(0.0), torch.nn.LayerNorm(hidden)

    def forward(self, hidden_states, input_tensor):
        return self.LayerNorm(self.dropout(self.dense(hidden_states)) + input_tensor)


def rewired(layer_norms=True, change=lambda norm: None):
    torch.manual_seed(0)
    model = torch.nn.Sequential(Output()).half().to(cuda()).eval()
    change(model[0].LayerNorm)
    sb = sten.SparsityBuilder()
    sb.set_weight("0.dense.weight", initial_sparsifier=sten.GroupedNMSparsifier(n=2, m=4, g=16), out_format=sten.GroupedNMTensor)
    model = sb.sparsify_model_inplace(model)
    assert sten.fuse_linear_epilogues(model, layer_norms=layer_norms) == 1
    return model[0]


@pytest.fixture
def replaced(monkeypatch):
    """How often the package's norm ran."""
    calls, real = [], sten.fusion.layer_norm
    monkeypatch.setattr(sten.fusion, "layer_norm", lambda *a, **k: calls.append(1) or real(*a, **k))
    return calls


def operands(hidden=64):
    gen = torch.Generator(device="cuda").manual_seed(1)
    return torch.randn(3, 128, 2 * hidden, device="cuda", generator=gen).half(), torch.randn(3, 128, hidden, device="cuda", generator=gen).half()


def run(mod):
    with torch.no_grad():
        return mod(*operands())


def test_a_plain_norm_is_replaced(replaced):
    ours = run(rewired())
    torchs = run(rewired(layer_norms=False))
    assert len(replaced) == 1 and ours.dtype == torch.float16
    # both compute in 32 bits and round once: a step of fp16 apart at most, where the two values before are on either side of a border
    assert bool(((ours.float() - torchs.float()).abs() <= 2.0 ** -10 * torchs.float().abs() + 2.0 ** -20).all())


def test_under_autocast_the_modules_own_norm_runs(replaced):
    with torch.autocast("cuda", dtype=torch.float16):
        ours, torchs = run(rewired()), run(rewired(layer_norms=False))
    assert not replaced and ours.dtype == torchs.dtype == torch.float32 and torch.equal(ours, torchs)
    with torch.autocast("cuda", enabled=False):
        run(rewired())
    assert len(replaced) == 1


def test_a_forward_of_the_instances_own_runs(replaced):
    def change(norm):
        norm.forward = lambda x, real=norm.forward: real(x) + 100
    ours, torchs = run(rewired(change=change)), run(rewired(layer_norms=False, change=change))
    assert not replaced and torch.equal(ours, torchs) and float(ours.float().min()) > 50


@pytest.mark.parametrize("kind", ["forward", "forward_pre", "module", "module_pre"])
def test_hooks_run(replaced, kind):
    mod, seen = rewired(), []

    def hook(m, *rest):
        if m is mod.LayerNorm:
            seen.append(1)
    register = {"forward": mod.LayerNorm.register_forward_hook, "forward_pre": mod.LayerNorm.register_forward_pre_hook,
                "module": torch.nn.modules.module.register_module_forward_hook, "module_pre": torch.nn.modules.module.register_module_forward_pre_hook}[kind]
    handle = register(hook)
    try:
        out = run(mod)
    finally:
        handle.remove()
    assert seen == [1] and not replaced and torch.equal(out, run(rewired(layer_norms=False)))


def test_norms_of_other_kinds_run_themselves(replaced):
    class Scaled(torch.nn.LayerNorm):
        def forward(self, x):
            return super().forward(x) * 2
    torchs = run(rewired(layer_norms=False))
    mod = rewired()
    norm = Scaled(64).half().to(cuda())
    norm.load_state_dict(mod.LayerNorm.state_dict())
    mod.LayerNorm = norm
    assert torch.equal(run(mod), torchs * 2) and not replaced


class Masked:
    """The smallest payload: whatever has a dense form."""

    def __init__(self, dense):
        self.dense, self.shape, self.dtype, self.device = dense, dense.shape, dense.dtype, dense.device

    def to_dense(self):
        return self.dense


def test_a_norm_of_sparse_parameters_runs_itself(replaced):
    """Through the dispatcher, as before."""
    outs = []
    for layer_norms in (False, True):
        mod = rewired(layer_norms)
        dense = mod.LayerNorm.weight.detach() * 3
        mod.LayerNorm.weight = sten.SparseParameterWrapper(sten.SparseTensorWrapper.wrapped_from_dense(Masked(dense), dense))
        outs.append(run(mod))
    assert torch.equal(*outs) and not replaced
