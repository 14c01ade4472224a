"""The enqueue-only op entry points captured into a CUDA graph as a process's
first calls (no eager call before: nothing is allocated or looked up in a way
that a capture forbids), replayed on new inputs, in a process of its own."""
import os
import subprocess
import sys

import pytest

from conftest import PKG, ROOT

pytestmark = pytest.mark.gpu

CODE = """
import torch, tpmd
F8 = torch.float8_e4m3fn
x, w = torch.randn(200, 512, device="cuda"), torch.randn(300, 512, device="cuda")
xq, wq = torch.empty(200, 512, dtype=F8, device="cuda"), torch.empty(300, 512, dtype=F8, device="cuda")
xs, ws = torch.empty(200, 4, device="cuda"), torch.empty(3, 4, device="cuda")
y = torch.empty(200, 300, device="cuda")
a = {t: [torch.randn(2, 90, 4, 64, device="cuda").to(t) for _ in range(3)] for t in (torch.float16, torch.float32)}
o = {t: torch.empty_like(a[t][0]) for t in a}
torch.cuda.synchronize()

def calls(st):
    tpmd.quant_f8(x, xq, xs, stream=st)
    tpmd.quant_f8(w, wq, ws, rows=128, stream=st)
    tpmd.gemm_f8(xq, xs, wq, ws, y, stream=st)
    for t in a:
        tpmd.attn_window(*a[t], o[t], 30, 5, 2, stream=st)

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls(torch.cuda.current_stream().cuda_stream)
for _ in range(2):
    for t in (x, w, *a[torch.float16], *a[torch.float32]):
        t.normal_()
    g.replay()
    torch.cuda.synchronize()
    got = [y.clone()] + [o[t].clone() for t in a]
    y.fill_(7.0)
    calls(0)
    tpmd.tpk_status()
    assert torch.equal(y, got[0])
    assert all(torch.equal(o[t], b) for t, b in zip(a, got[1:]))
print("captured and replayed")
"""


def test_first_calls_are_captured():
    r = subprocess.run([sys.executable, "-c", CODE], capture_output=True, text=True, timeout=300, cwd=ROOT,
                       env=dict(os.environ, PYTHONPATH=PKG))
    assert r.returncode == 0 and "captured and replayed" in r.stdout, r.stdout + r.stderr
