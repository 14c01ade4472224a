"""Ops that follow one another on a stream without a pause, each a
programmatic dependent of the one ahead: scales, rows, biases and lengths
that the call ahead writes, against the same calls with a synchronise after
each. The same kernels on the same inputs: equal bit for bit."""
import pytest
import torch

import tpmd

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _f8(M, K):
    return torch.empty(M, -(-K // 16) * 16, dtype=F8, device="cuda")[:, :K], torch.empty(M, -(-K // 128), device="cuda")


def _weight(N, K, gen):
    w = torch.randn(N, K, generator=gen, device="cuda") / K ** 0.5
    q = torch.empty(N, -(-K // 16) * 16, dtype=F8, device="cuda")[:, :K]
    s = torch.empty(-(-N // 128), -(-K // 128), device="cuda")
    return tpmd.quant_f8(w, q, s, rows=128)


@pytest.mark.parametrize("M,H,F", [(1, 256, 512), (180, 1024, 4096), (2600, 512, 2048)])
def test_quantise_multiply_chain(M, H, F):
    """x -> 8 bits -> product in 8 bits with its scales -> product -> x, over
    and over: every call's scales come from the call ahead"""
    g = torch.Generator(device="cuda").manual_seed(M)
    w1, w2 = _weight(F, H, g), _weight(H, F, g)
    bias = 0.1 * torch.randn(F, generator=g, device="cuda")
    x0 = torch.randn(M, H, generator=g, device="cuda") * torch.exp(torch.randn(M, 1, generator=g, device="cuda"))

    def run(steps, pause):
        x, seen = x0.clone(), []
        xq, xs = _f8(M, H)
        hq, hs = _f8(M, F)
        for i in range(steps):
            tpmd.quant_f8(x, xq, xs)
            pause()
            tpmd.gemm_f8(xq, xs, *w1, hq, sy=hs, bias=bias, act=2)
            pause()
            y = torch.empty_like(x)
            tpmd.gemm_f8(hq, hs, *w2, y)
            pause()
            # rows of other sizes from step to step: a stale scale shows
            x = y * (1.0 + 3.0 * (i % 3))
            seen.append(y)
        return seen

    want = run(12, torch.cuda.synchronize)
    torch.cuda.synchronize()
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(run(12, lambda: None), want))
    tpmd.tpk_status()


def test_a_product_gives_the_next_one_its_bias():
    """tpk_gemm_f8's f32 output row as the bias of the call behind it, and a
    quantisation of that call's output"""
    g = torch.Generator(device="cuda").manual_seed(1)
    K, N = 256, 384
    w = _weight(N, K, g)
    rows = [torch.randn(m, K, generator=g, device="cuda") for m in (1, 1, 1, 60)]
    qs = [tpmd.quant_f8(r, *_f8(*r.shape)) for r in rows]

    def run(pause):
        out = []
        for i in range(9):
            row, y = torch.empty(1, N, device="cuda"), torch.empty(60, N, device="cuda")
            yq, ys = _f8(60, N)
            tpmd.gemm_f8(*qs[i % 3], *w, row)
            pause()
            tpmd.gemm_f8(*qs[3], *w, y, bias=row.view(N))
            pause()
            tpmd.quant_f8(y, yq, ys)
            out += [y, yq.float(), ys]
        return out

    want = run(torch.cuda.synchronize)
    torch.cuda.synchronize()
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(run(lambda: None), want))
    tpmd.tpk_status()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_lengths_and_rows_written_just_ahead(dtype):
    """a growing cache: the lengths and the new token's rows are written by
    the kernels right ahead of the attention that reads them"""
    g = torch.Generator(device="cuda").manual_seed(2)
    B, T, Hq, Hkv, D = 5, 300, 8, 2, 64
    new = torch.randn(40, 3, B, 1, Hq, D, generator=g, device="cuda").to(dtype)

    def run(pause):
        k, v = (torch.full((B, T, Hkv, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        n = torch.tensor([0, 7, 100, 200, 259], dtype=torch.int32, device="cuda")
        start, out = n.clone().long(), []
        k[torch.arange(T, device="cuda")[None] < n[:, None]] = 0.25
        v[torch.arange(T, device="cuda")[None] < n[:, None]] = 0.5
        at = torch.arange(B, device="cuda")
        for t in range(40):
            q, kk, vv = new[t]
            k[at, start + t] = kk[:, 0, :Hkv]
            v[at, start + t] = vv[:, 0, :Hkv]
            n.add_(1)
            pause()
            o = torch.empty(B, 1, Hq, D, dtype=dtype, device="cuda")
            tpmd.attn_window(q, k, v, o, 90, 0, 3, kv_len=n)
            pause()
            out.append(o)
        return out

    want = run(torch.cuda.synchronize)
    torch.cuda.synchronize()
    assert not any(bool(o.isnan().any()) for o in want)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(lambda: None), want))
    tpmd.tpk_status()
