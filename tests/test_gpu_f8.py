"""8-bit quantisation (tpk_quant_f8) and the block-scaled 8-bit product
(tpk_gemm_f8) against their definitions.

* The quantiser's scales and bytes are IEEE float32 arithmetic and one
  rounding to e4m3: equal, bit for bit, to the same steps on the CPU.
* The product against float64: with S = sum_b sx sw sum_k |x w|, an f32 sum
  of 128 products per block (exact products, each addition off by at most
  2^-23 relative whichever way it rounds), one product of scales, one
  multiply-add per block and the bias: |err| <= (128 + 3 blocks + 2) 2^-23
  (S + |bias|). The activations change an error by a factor below 1.13 and
  add a few ulp (2^-21 of |v| and of 1). An f16 output adds 2^-11 |y| (2^-25
  below the normal range).
* The 8-bit output equals tpk_quant_f8 of the f32 output, bit for bit: the
  same sums, the same quantisation.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import tpmd

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def quant_ref(x, rows):
    """(bytes as float8, scales) of a CPU tensor, float32 step by step"""
    M, K = x.shape
    x = x.float()
    mb, kb = -(-M // rows), -(-K // 128)
    full = torch.zeros(mb * rows, kb * 128)
    full[:M, :K] = x
    b = full.view(mb, rows, kb, 128)
    a = torch.nan_to_num(b.abs(), nan=0.0, posinf=float("inf")).amax(dim=(1, 3))
    s = torch.maximum(a / torch.full_like(a, 448.0), torch.full_like(a, 2.0 ** -126))
    v = (b / s[:, None, :, None]).reshape(mb * rows, kb * 128)[:M, :K]
    return v.clamp(-448.0, 448.0).to(F8), s


def padded(M, K, dtype=F8, extra=0):
    """[M, K] view with 16-byte rows, poisoned between them"""
    ld = -(-K // 16) * 16 + extra
    t = torch.full((M, ld), 0x7F, dtype=torch.uint8, device="cuda")
    return t.view(dtype)[:, :K], t


def quantised(M, K, rows, gen, scale=1.0):
    x = torch.randn(M, K, generator=gen) * scale * torch.exp(torch.randn(M, 1, generator=gen))
    q, s = quant_ref(x, rows)
    d, _ = padded(M, K)
    d.copy_(q)
    return d, s.cuda()


def same_bytes(a, b):
    """equal e4m3 values; NaN equals NaN whatever its sign"""
    a, b = a.cpu().float(), b.cpu().float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 129), (180, 1024), (127, 40), (129, 300), (256, 128), (5, 8), (700, 1000)])
def test_quant(M, K, dtype, rows):
    g = torch.Generator().manual_seed(M * 1000 + K + rows)
    x = (torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(M, K, generator=g))).to(dtype)
    q, raw = padded(M, K)
    s = torch.zeros(-(-M // rows), -(-K // 128), device="cuda")
    tpmd.quant_f8(x.cuda(), q, s, rows=rows)
    rq, rs = quant_ref(x, rows)
    assert torch.equal(s.cpu(), rs)
    assert same_bytes(q, rq)
    assert bool((raw[:, K:] == 0x7F).all())  # nothing written between rows


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_quant_strides_and_alignment(dtype, rows):
    """rows that start anywhere: column slices at odd offsets, padded scales"""
    g = torch.Generator().manual_seed(3)
    big = torch.randn(131, 517, generator=g).to(dtype)
    for c0, K in ((1, 300), (3, 128), (8, 257), (0, 515)):
        x = big.cuda()[:, c0:c0 + K]
        raw = torch.full((131, 601), 0x55, dtype=torch.uint8, device="cuda")
        q = raw.view(F8)[:, 7:7 + K]
        sraw = torch.full((131, 9), -1.0, device="cuda")
        s = sraw[:-(-131 // rows), 2:2 - (-K // 128)]
        tpmd.quant_f8(x, q, s, rows=rows)
        rq, rs = quant_ref(big[:, c0:c0 + K], rows)
        assert torch.equal(s.cpu(), rs) and same_bytes(q, rq)
        assert bool((raw[:, :7] == 0x55).all()) and bool((raw[:, 7 + K:] == 0x55).all())
        assert bool((sraw[:, :2] == -1).all()) and bool((sraw[:, 2 - (-K // 128):] == -1).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows", [1, 128])
def test_quant_special_values(rows, dtype):
    """zeros, the smallest and largest numbers, infinities, NaN, ties"""
    x = torch.zeros(130, 640)
    x[0, 0:128] = 1e-45
    x[1, 128:256] = 3.4e38
    x[2, 256] = float("inf")
    x[2, 257] = -3.0
    x[3, 384] = float("nan")
    x[3, 385] = 2.0
    x[4, 512:528] = torch.tensor([448.0, 1.0625, 1.1875, 17.0, 19.0, -1.0625, 2 ** -10, 3 * 2.0 ** -10] * 2)
    x = x.to(dtype)
    q, _ = padded(130, 640)
    s = torch.zeros(-(-130 // rows), 5, device="cuda")
    tpmd.quant_f8(x.cuda(), q, s, rows=rows)
    rq, rs = quant_ref(x, rows)
    assert torch.equal(s.cpu(), rs) and same_bytes(q, rq)


def gemm_ref(X, sx, W, sw, bias, act):
    """(y, bound) in float64"""
    (M, K), N = X.shape, W.shape[0]
    X, W, sx, sw = X.cpu().double(), W.cpu().double(), sx.cpu().double(), sw.cpu().double()
    y, S = torch.zeros(M, N, dtype=torch.float64), torch.zeros(M, N, dtype=torch.float64)
    kb = -(-K // 128)
    for b in range(kb):
        c = slice(b * 128, b * 128 + 128)
        f = sx[:, b:b + 1] * sw[:, b].repeat_interleave(128)[None, :N]
        y += X[:, c] @ W[:, c].t() * f
        S += X[:, c].abs() @ W[:, c].abs().t() * f
    if bias is not None:
        y, S = y + bias.cpu().double(), S + bias.cpu().double().abs()
    bound = (128 + 3 * kb + 2) * 2.0 ** -23 * S
    if act:
        bound = 1.13 * bound + 2.0 ** -21 * (y.abs() + 1)
    if act == 1:
        y = torch.nn.functional.gelu(y)
    elif act == 2:
        y = torch.nn.functional.gelu(y, approximate="tanh")
    elif act == 3:
        y = torch.nn.functional.leaky_relu(y, 0.2)
    return y, bound


def run_gemm(M, N, K, out, act=0, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed + M + 3 * N + 7 * K)
    X, sx = quantised(M, K, 1, g)
    W, sw = quantised(N, K, 128, g, scale=K ** -0.5)
    b = torch.randn(N, generator=g).cuda() if bias else None
    Y = torch.full((M, N), float("nan"), dtype=out, device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, Y, bias=b, act=act)
    tpmd.tpk_status()
    return (X, sx, W, sw, b), Y


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 1024, 1024), (2, 130, 257), (60, 1024, 512), (128, 128, 4096), (129, 129, 129),
          (180, 1024, 1024), (180, 1024, 4096), (180, 4096, 1024), (257, 264, 40), (777, 1000, 528), (1000, 2048, 768),
          (3000, 640, 1024), (64, 8192, 1024), (5000, 1100, 400), (2500, 2050, 256), (19000, 200, 130)]


@pytest.mark.parametrize("out", [torch.float32, torch.float16])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm(M, N, K, out):
    a, Y = run_gemm(M, N, K, out, bias=M % 2 == 0)
    y, bound = gemm_ref(*a, 0)
    if out == torch.float16:
        bound = bound + 2.0 ** -11 * y.abs() + 2.0 ** -25
    err = (Y.cpu().double() - y).abs()
    worst = float((err / (bound + 1e-300)).max())
    print(f"{M}x{N}x{K}: worst err / bound {worst:.3f}")
    assert worst <= 1.0


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("M,N,K", [(180, 1024, 1024), (50, 200, 4096), (700, 3000, 384), (4100, 1300, 140)])
def test_gemm_activations(M, N, K, act):
    a, Y = run_gemm(M, N, K, torch.float32, act=act)
    y, bound = gemm_ref(*a, act)
    assert bool(((Y.cpu().double() - y).abs() <= bound).all())


@pytest.mark.parametrize("act", [0, 2])
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 1024, 1024), (180, 4096, 1024), (130, 200, 300), (777, 1000, 528),
                                   (60, 130, 4096), (3000, 640, 256), (5000, 1100, 144)])
def test_gemm_f8_output_is_the_quantised_f32_output(M, N, K, act):
    (X, sx, W, sw, b), Y = run_gemm(M, N, K, torch.float32, act=act)
    q, raw = padded(M, N, extra=16)
    sy = torch.zeros(M, -(-N // 128), device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, q, sy=sy, bias=b, act=act)
    rq, rs = quant_ref(Y.cpu(), 1)
    assert torch.equal(sy.cpu(), rs) and same_bytes(q, rq)
    assert bool((raw[:, N:] == 0x7F).all())


def test_gemm_output_strides():
    """rows of Y, sx and sw with strides of their own, Y not 16-byte aligned"""
    g = torch.Generator().manual_seed(1)
    M, N, K = 150, 190, 300
    X, sx = quantised(M, K, 1, g)
    W, sw = quantised(N, K, 128, g)
    want = torch.empty(M, N, device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, want)
    sx2, sw2 = torch.zeros(M, 11, device="cuda"), torch.zeros(2, 7, device="cuda")
    sx2[:, 4:7], sw2[:, 1:4] = sx, sw
    for dt, off in ((torch.float32, 1), (torch.float16, 3), (torch.float32, 4)):
        big = torch.full((M, 233), 7.0, dtype=dt, device="cuda")
        tpmd.gemm_f8(X, sx2[:, 4:7], W, sw2[:, 1:4], big[:, off:off + N])
        assert torch.equal(big[:, off:off + N], want.to(dt))
        assert bool((big[:, :off] == 7).all()) and bool((big[:, off + N:] == 7).all())


# 128 x 128 and 256 x 256 tiles
@pytest.mark.parametrize("M,N", [(131, 131), (300, 257), (2310, 2317), (2400, 2306)])
@pytest.mark.parametrize("out", [torch.float32, torch.float16, F8])
def test_gemm_rows_off_vector_boundaries(M, N, out):
    """the same bytes as with aligned rows, and none beside them"""
    K = 72
    g = torch.Generator().manual_seed(M + N)
    (x, sx), (w, sw) = quantised(M, K, 1, g), quantised(N, K, 128, g)
    bias = torch.randn(N, generator=g).cuda()
    nb, es = -(-N // 128), out.itemsize
    ld = -(-N // 16) * 16
    want = torch.zeros(M, ld * es, dtype=torch.uint8, device="cuda").view(out)[:, :N]
    scales = [torch.zeros(M, nb, device="cuda") if out is F8 else None for _ in range(2)]
    tpmd.gemm_f8(x, sx, w, sw, want, sy=scales[0], bias=bias, act=1)
    for ld, at in ((N, 0), (N + 5, 0), (N + 1, 3)):
        raw = torch.full(((M * ld + at) * es,), 0x55, dtype=torch.uint8, device="cuda")
        y = raw[at * es:].view(out).view(M, ld)[:, :N]
        tpmd.gemm_f8(x, sx, w, sw, y, sy=scales[1], bias=bias, act=1)
        tpmd.tpk_status()
        assert torch.equal(y.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))
        assert out is not F8 or torch.equal(*scales)
        beside = raw[at * es:].view(M, ld * es)[:, N * es:]
        assert bool((beside == 0x55).all()) and bool((raw[:at * es] == 0x55).all())


@pytest.mark.parametrize("rows", [1, 128])
def test_quant_blocks_of_zeros(rows):
    """the smallest scale; a NaN between the zeros stays one"""
    x = torch.zeros(200, 333)
    x[3, 7], x[3, 8], x[150, 200] = float("nan"), -0.0, 1.5
    for dt in (torch.float32, torch.float16):
        q, _ = padded(200, 333)
        s = torch.zeros(-(-200 // rows), 3, device="cuda")
        tpmd.quant_f8(x.to(dt).cuda(), q, s, rows=rows)
        rq, rs = quant_ref(x, rows)
        assert torch.equal(s.cpu(), rs) and same_bytes(q, rq)


def test_gemm_special_scales():
    """negative, zero, infinite and NaN scales and NaN bytes go where the
    formula takes them; the rows beside them are not touched"""
    g = torch.Generator().manual_seed(2)
    X, sx = quantised(40, 256, 1, g)
    W, sw = quantised(130, 256, 128, g)
    want = torch.empty(40, 130, device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, want)
    sx[3] = -sx[3]
    sx[5, 1] = float("nan")
    sx[7] = 0.0
    X.view(torch.uint8)[9, 200] = 0x7F
    Y = torch.empty(40, 130, device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, Y)
    assert torch.equal(Y[3], -want[3]) and bool(Y[5].isnan().all()) and bool((Y[7] == 0).all())
    assert bool(Y[9].isnan().all())
    rest = [i for i in range(40) if i not in (3, 5, 7, 9)]
    assert torch.equal(Y[rest], want[rest])


def test_gemm_repeats_streams_and_graphs():
    """same bits on every call, on two streams at once, and from a captured
    graph replayed on new inputs"""
    g = torch.Generator().manual_seed(4)
    ins = [(quantised(180, 4096, 1, g), quantised(1024, 4096, 128, g)) for _ in range(2)]
    want = []
    for (X, sx), (W, sw) in ins:
        Y = torch.empty(180, 1024, device="cuda")
        tpmd.gemm_f8(X, sx, W, sw, Y)
        want.append(Y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    outs = [[torch.empty(180, 1024, device="cuda") for _ in range(8)] for _ in ins]
    torch.cuda.synchronize()
    for r in range(8):
        for i, ((X, sx), (W, sw)) in enumerate(ins):
            tpmd.gemm_f8(X, sx, W, sw, outs[i][r], stream=streams[i].cuda_stream)
    for i, st in enumerate(streams):
        tpmd.tpk_status(st.cuda_stream)
        assert all(torch.equal(o, want[i]) for o in outs[i])
    (X, sx), (W, sw) = (tuple(t.clone() for t in p) for p in ins[0])
    x16 = torch.randn(180, 4096, generator=g).cuda()
    Y = torch.empty(180, 1024, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        tpmd.quant_f8(x16, X, sx, stream=st)
        tpmd.gemm_f8(X, sx, W, sw, Y, stream=st)
    for _ in range(3):
        x16.copy_(torch.randn(180, 4096, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        q, s = padded(180, 4096)[0], torch.empty_like(sx)
        tpmd.quant_f8(x16, q, s)
        ref = torch.empty_like(Y)
        tpmd.gemm_f8(q, s, W, sw, ref)
        assert torch.equal(Y, ref)


def test_linear_from_float32():
    """quantise, multiply, quantise in the epilogue, multiply: an MLP as the
    sampler would run it, against float64 on the unquantised numbers. Each
    quantisation is off by at most 2^-4 of an element or 2^-10 of its
    block's scale, and the scale is 1/448 of the block's maximum: the bound
    carries these through both products."""
    g = torch.Generator().manual_seed(5)
    M, H, F = 180, 256, 1024
    x = torch.randn(M, H, generator=g)
    w1, w2 = torch.randn(F, H, generator=g) / H ** 0.5, torch.randn(H, F, generator=g) / F ** 0.5

    def dev(t, rows):
        q = torch.empty(t.shape, dtype=F8, device="cuda")
        s = torch.empty(-(-t.shape[0] // rows), -(-t.shape[1] // 128), device="cuda")
        return tpmd.quant_f8(t.cuda(), q, s, rows=rows)

    (xq, xs), (w1q, w1s), (w2q, w2s) = dev(x, 1), dev(w1, 128), dev(w2, 128)
    hq, hs = torch.empty(M, F, dtype=F8, device="cuda"), torch.empty(M, F // 128, device="cuda")
    y = torch.empty(M, H, device="cuda")
    tpmd.gemm_f8(xq, xs, w1q, w1s, hq, sy=hs, act=2)
    tpmd.gemm_f8(hq, hs, w2q, w2s, y)
    tpmd.tpk_status()

    def off(t, s, rows):  # largest distance of a quantised element from its own
        step = s.cpu().double().repeat_interleave(rows, 0)[:t.shape[0]].repeat_interleave(128, 1)[:, :t.shape[1]]
        return torch.maximum(t.abs() * 2.0 ** -4, step * 2.0 ** -10)

    x, w1, w2 = x.double(), w1.double(), w2.double()
    pre = x @ w1.t()
    h = torch.nn.functional.gelu(pre, approximate="tanh")
    dx, dw1, dw2 = off(x, xs, 1), off(w1, w1s, 128), off(w2, w2s, 128)
    dpre = dx @ w1.abs().t() + (x.abs() + dx) @ dw1.t()
    dh = 1.13 * dpre
    dh = dh + torch.maximum((h.abs() + dh) * 2.0 ** -4, hs.cpu().double().repeat_interleave(128, 1) * 2.0 ** -10)
    bound = dh @ w2.abs().t() + (h.abs() + dh) @ dw2.t()
    err = (y.cpu().double() - h @ w2.t()).abs()
    assert bool((err <= bound * (1 + 1e-4) + 1e-5).all())
    # rounding errors of either sign: far inside the worst case
    assert float(err.norm() / (h @ w2.t()).norm()) < 3 * 2.0 ** -4
