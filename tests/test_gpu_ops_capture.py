"""The enqueue-only op entry points captured into a CUDA graph as a process's
first calls (no eager call before: nothing is allocated or looked up in a way
that a capture forbids), replayed on new inputs, in a process of its own."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import tpmd
from conftest import PKG, ROOT

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn

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


def _ops():
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w = torch.randn(200, 512, device="cuda", generator=g), torch.randn(300, 512, device="cuda", generator=g)
    xq, wq = torch.empty(200, 512, dtype=F8, device="cuda"), torch.empty(300, 512, dtype=F8, device="cuda")
    xs, ws, y = torch.empty(200, 4, device="cuda"), torch.empty(3, 4, device="cuda"), torch.empty(200, 300, device="cuda")
    q = torch.randn(2, 50, 4, 64, device="cuda", generator=g)
    o = {t: torch.empty_like(q, dtype=t) for t in (torch.float16, torch.float32)}

    def run(st):
        tpmd.quant_f8(x, xq, xs, stream=st)
        tpmd.quant_f8(w, wq, ws, rows=128, stream=st)
        tpmd.gemm_f8(xq, xs, wq, ws, y, stream=st)
        for t in o:
            z = q if t is q.dtype else q16
            tpmd.attn_window(z, z, z, o[t], 20, 3, 2, stream=st)
    q16 = q.half()
    return x, q, q16, [y, *o.values()], run


def test_captured_behind_copies_fills_and_other_streams():
    """an op is the dependent of whatever node comes before it: a copy, a
    fill, two streams that join, a kernel of another library"""
    x, q, q16, outs, run = _ops()
    new, side = torch.empty_like(x), torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        x.copy_(new)  # a copy node
        run(main.cuda_stream)
        for t in outs:
            t.zero_()  # a fill node; the ops write everything again
        side.wait_stream(main)
        with torch.cuda.stream(side):
            q.mul_(0.5)
            q16.copy_(q)
            tpmd.attn_window(q, q, q, outs[2], 20, 3, 2, stream=side.cuda_stream)
        x.mul_(2.0)
        main.wait_stream(side)  # two nodes before the first op
        run(main.cuda_stream)
    start = q.clone()
    for i in range(3):
        new.normal_()
        q.copy_(start)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert torch.equal(x, new * 2) and torch.equal(q, start * 0.5)
        for t in outs:
            t.fill_(9.0)
        run(0)
        tpmd.tpk_status()
        assert all(torch.equal(a, b) for a, b in zip(outs, got))


def test_two_host_threads():
    """calls from two threads at once, each on a stream of its own"""
    sets = [_ops() for _ in range(2)]
    want = []
    for s in sets:
        s[4](0)
        torch.cuda.synchronize()
        want.append([t.clone() for t in s[3]])
    bad = []

    def work(i):
        try:
            st = torch.cuda.Stream()
            for _ in range(40):
                sets[i][4](st.cuda_stream)
                tpmd.tpk_status(st.cuda_stream)
                if not all(torch.equal(a, b) for a, b in zip(sets[i][3], want[i])):
                    bad.append(i)
        except Exception as e:  # noqa: BLE001 (reported below)
            bad.append(repr(e))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
