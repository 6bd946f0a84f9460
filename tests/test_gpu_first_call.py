"""An operator's first call in a process, which loads its kernels, inside a stream capture."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attention-cpu_amd")
CODE = """
import torch
import flash_attention_amd as fa
q = torch.randn(1, 4, 300, 64, device="cuda").bfloat16()
out = torch.empty_like(q)
cfg = fa.score_config(fa.DTYPE_BF16, 1, 4, 4, 300, 300, 64, causal=True)

def call():
    p = q.data_ptr()
    fa.score_attention_device(cfg, p, p, p, out.data_ptr(), 0, torch.cuda.current_stream().cuda_stream)

side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    call()
for _ in range(3):
    q.normal_()
    out.fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    got = out.clone()
    call()
    torch.cuda.synchronize()
    assert torch.equal(got, out) and torch.isfinite(got).all()
print("same")
"""


def test_first_call_in_a_capture():
    r = subprocess.run([sys.executable, "-c", CODE], capture_output=True, text=True, timeout=100,
                       env=dict(os.environ, PYTHONPATH=PKG))
    assert r.stdout.strip().endswith("same"), (r.stdout, r.stderr[-2000:])
