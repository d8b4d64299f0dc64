"""The first call of an operator in a process, made while a stream is captured: its set-up happens then, and the graph gives
what an eager call gives. One process each, since an operator is set up once per device."""

from __future__ import annotations

import subprocess
import sys

import pytest

from .conftest import ROOT, cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a B200")]

PROGRAM = """
import torch
from selas_b200 import _lib, ops

_lib.lib()
x = torch.randn(300, 512, device="cuda")
h, w = x.bfloat16(), torch.randn(2048, 512, device="cuda").bfloat16()
ids = torch.arange(300, device="cuda")[:, None]
call = {
    "layer_norm": lambda: (ops.layer_norm(x),),
    "layer_norm_backward": lambda: ops.layer_norm_backward(x, x),
    "rope_axes": lambda: (ops.rope_axes(x.view(1, 4, 300, 128), ids, (128,)),),
    "linear_act": lambda: (ops.linear_act(h, w, None, "gelu"),),
}[NAME]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = call()
graph.replay()
assert all(torch.equal(a, b) for a, b in zip(out, call()))
torch.cuda.synchronize()
assert _lib.device_status() == 0
"""


@pytest.mark.parametrize("name", ["layer_norm", "layer_norm_backward", "rope_axes", "linear_act"])
def test_first_call_is_captured(name):
    r = subprocess.run([sys.executable, "-c", PROGRAM.replace("NAME", repr(name))], cwd=ROOT, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stdout + r.stderr
