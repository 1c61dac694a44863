"""A library call that fails in a backward pass, on one of autograd's threads, is a RuntimeError: not the end of the process."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu
CALLS = {"nmg_layer_norm_backward": "sten.layer_norm(x)", "nmg_embedding_backward": "sten.embedding(ids, x)", "nmg_token_log_probs_backward": "sten.token_log_probs(x).entropy",
         "nmg_distill_backward": "sten.distillation_loss(x, ids[:, None], lp, reduction='none')"}


def test_failing_library_calls(tmp_path):
    stub = tmp_path / "stub.c"  # takes the place of the library's functions
    stub.write_text("".join(f"int {name}(void) {{ return 3; }}\n" for name in CALLS))
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(tmp_path / "stub.so"), str(stub)], check=True)
    lines = ["import torch, sten_b200 as sten", "x = torch.randn(3, 64, device='cuda', requires_grad=True)", "ids, lp = torch.arange(3, device='cuda'), torch.zeros(3, 1, device='cuda')"]
    for call in CALLS.values():
        lines += [f"y = {call}.sum()", "try:", "    torch.autograd.grad(y, x)", "except RuntimeError as e:", "    print('told:', 'nmg_b200 status 3' in str(e))"]
    env = {**os.environ, "LD_PRELOAD": str(tmp_path / "stub.so"), "PYTHONPATH": ROOT}
    r = subprocess.run([sys.executable, "-c", "\n".join(lines)], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.count("told: True") == len(CALLS), (r.returncode, r.stdout[-500:], r.stderr[-2000:])
