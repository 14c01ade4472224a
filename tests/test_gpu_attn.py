"""Sliding-window attention (tpk_attn_window) against its formula in float64.

Bound per output element, with p the float64 softmax weights, A = sum_j p_j
|v_j| and x = largest scale sum_d |q_d k_d| of the row:
* a score is an f32 sum of D products, scaled and shifted by the maximum:
  off by at most d = (D + 4) 2^-23 x, so a weight by 2 d relative (numerator
  and normaliser), plus 2^-20 for exponentials and 2^-23 per key for the sums;
* f16: weights may be rounded to f16 on their way into the product with v
  (2^-11 relative, 2^-25 absolute per key below the normal range, against a
  largest weight of 1 or more), the output once more (2^-11 |o|, 2^-25).
"""
from __future__ import annotations

import pytest
import torch

import tpmd

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16}


def reference(q, k, v, left, right, sinks, scale, q_len=None, kv_len=None):
    """(out, bound, rows that exist) in float64 on the CPU"""
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1:3]
    f16 = q.dtype == torch.float16
    out = torch.zeros(B, Tq, Hq, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    rows = torch.zeros(B, Tq, dtype=torch.bool)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    for b in range(B):
        n = Tq if q_len is None else min(max(int(q_len[b]), 0), Tq)
        L = Tk if kv_len is None else min(max(int(kv_len[b]), 0), Tk)
        rows[b, :n] = True
        if n == 0 or L == 0:
            continue
        p = torch.arange(n)[:, None] + L - n
        j = torch.arange(L)[None, :]
        ok = torch.ones(n, L, dtype=torch.bool)
        if right >= 0:
            ok &= j <= p + right
        if left >= 0:
            ok &= (j >= p - left) | (j < sinks)
        seen = ok.any(dim=1)
        for h in range(Hq):
            kk, vv, qq = k[b, :L, h // (Hq // Hkv)], v[b, :L, h // (Hq // Hkv)], q[b, :n, h]
            # rows and columns that nobody looks at may hold anything
            kk = torch.where(ok.any(dim=0)[:, None], kk, torch.zeros_like(kk))
            vv = torch.where(ok.any(dim=0)[:, None], vv, torch.zeros_like(vv))
            s = (qq @ kk.t() * scale).masked_fill(~ok, -float("inf"))
            w = torch.softmax(s, dim=1)
            w = torch.where(seen[:, None], w, torch.zeros_like(w))
            o, A = w @ vv, w @ vv.abs()
            x = (qq.abs() @ kk.abs().t() * abs(scale)).masked_fill(~ok, 0).amax(dim=1, keepdim=True)
            keys = ok.sum(dim=1, keepdim=True)
            e = A * (2 * (D + 4) * 2.0 ** -23 * x + 2.0 ** -20 + keys * 2.0 ** -23) + 2.0 ** -24 * o.abs() + 1e-37
            if f16:
                # the largest weight (1 / normaliser) is at least 1 / keys of their sum
                top = w.amax(dim=1, keepdim=True)
                e = e + 2.0 ** -11 * A + keys * 2.0 ** -25 * top * vv.abs().max() + 2.0 ** -11 * o.abs() + 2.0 ** -25
            out[b, :n, h], bound[b, :n, h] = o, e
    return out, bound, rows


def check(q, k, v, left, right=0, sinks=0, scale=None, q_len=None, kv_len=None, out=None, stream=0):
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    out.fill_(77.0)
    torch.cuda.synchronize()
    tpmd.attn_window(q, k, v, out, left, right, sinks, scale=scale, q_len=q_len, kv_len=kv_len, stream=stream)
    tpmd.tpk_status(stream)
    ref, bound, rows = reference(q, k, v, left, right, sinks, q.shape[3] ** -0.5 if scale is None else scale, q_len, kv_len)
    got = out.cpu().double()
    assert bool((got[~rows] == 77.0).all())  # rows behind a sequence's end are left
    err = (got[rows] - ref[rows]).abs()
    assert not bool(got[rows].isnan().any())
    # (rows that see nothing: zeros, with a bound of zero)
    assert bool((err <= bound[rows]).all()), float((err / bound[rows].clamp(min=1e-37)).max())
    return out


def make(B, Tq, Tk, Hq, Hkv, D, dtype, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed * 7 + B + Tq + Tk + Hq + D)
    t = [torch.randn(B, T, H, D, generator=g) * s for T, H, s in ((Tq, Hq, gain), (Tk, Hkv, 1.0), (Tk, Hkv, 1.0))]
    return [x.to(TYPES[dtype]).cuda() for x in t]


def lens(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# B, Tq, Tk, Hq, Hkv, D, left, right, sinks
SHAPES = [
    (1, 1, 1, 1, 1, 64, 0, 0, 0), (1, 1, 1, 1, 1, 1, -1, -1, 0), (2, 1, 5, 4, 2, 64, 2, 0, 1),
    (3, 60, 60, 8, 8, 128, 2, 2, 10), (3, 60, 60, 4, 4, 64, 7, 7, 0), (1, 128, 128, 2, 1, 128, 31, 0, 0),
    (1, 129, 129, 2, 2, 64, -1, 0, 0), (1, 127, 127, 3, 1, 32, 5, -1, 4), (2, 300, 300, 6, 2, 80, 40, 0, 3),
    (1, 513, 513, 4, 4, 128, 127, 0, 130), (1, 700, 700, 2, 1, 96, 128, 64, 128), (1, 257, 600, 5, 1, 40, 200, 0, 7),
    (2, 1, 1000, 8, 1, 128, 255, 0, 4), (1, 1, 4097, 8, 2, 64, -1, 0, 0), (4, 3, 640, 6, 3, 128, 100, 0, 2),
    (1, 2, 333, 16, 2, 128, 0, 0, 0), (1, 5, 2000, 12, 12, 64, -1, 0, 0), (1, 40, 40, 2, 2, 256, 9, 3, 1),
    (1, 100, 100, 2, 2, 160, 20, 0, 5), (1, 64, 64, 130, 1, 16, 10, 0, 1), (1, 1000, 1000, 1, 1, 64, 0, 0, 0),
    (1, 333, 333, 7, 1, 72, 50, 20, 200), (1, 1025, 1025, 2, 2, 128, 256, 256, 0), (1, 90, 900, 2, 2, 128, -1, -1, 0)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("case", SHAPES, ids=lambda c: "-".join(map(str, c)))
def test_shapes(case, dtype):
    B, Tq, Tk, Hq, Hkv, D, left, right, sinks = case
    check(*make(B, Tq, Tk, Hq, Hkv, D, dtype), left, right, sinks)


# many rows: enough work for every SM without sharing out keys
MANY = [(8, 600, 600, 12, 6, 64, 99, 0, 3), (3, 1300, 1300, 40, 10, 128, 200, 31, 140), (2, 2049, 2049, 16, 16, 80, 64, 0, 1),
        (40, 250, 300, 12, 4, 128, -1, 0, 0), (1, 2000, 2000, 30, 30, 32, 3, 3, 5), (4, 515, 515, 100, 20, 40, 0, -1, 2),
        (150, 1, 700, 4, 2, 128, 300, 0, 4), (160, 3, 200, 2, 1, 64, -1, 0, 0)]


@pytest.mark.parametrize("case", MANY, ids=lambda c: "-".join(map(str, c)))
def test_many_rows(case):
    B, Tq, Tk, Hq, Hkv, D, left, right, sinks = case
    q, k, v = make(B, Tq, Tk, Hq, Hkv, D, "f16", gain=3.0)
    check(q, k, v, left, right, sinks)
    # lengths of their own; NaN and infinities behind the ends
    n = lens(*[Tq * (7 * i % (B + 1)) // B for i in range(B)])
    L = lens(*[x if Tq == Tk else max(x, Tk * (5 * i % (B + 1)) // B) for i, x in enumerate(n.tolist())])
    for b, x in enumerate(L.tolist()):
        k[b, x:], v[b, x:] = float("nan"), float("inf")
    check(q, k, v, left, right, sinks, q_len=n, kv_len=L)


# f32 rows: one to sixteen a CTA, every width of a lane's share, one sequence and hundreds
F32_ROWS = [(1, 1, 300, 4, 1, 32, 70, 0, 3), (2, 2, 301, 4, 1, 20, -1, 0, 0), (1, 4, 77, 4, 1, 128, 20, 5, 9),
            (1, 3, 500, 3, 1, 96, 50, 0, 9), (3, 30, 95, 2, 2, 33, 12, 2, 17), (1, 9, 1100, 3, 1, 200, 333, 0, 130),
            (2, 1, 640, 4, 2, 256, -1, 0, 0), (1, 31, 31, 2, 1, 250, 8, 0, 2), (80, 1, 70, 4, 4, 128, 40, 0, 3),
            (100, 2, 50, 9, 3, 64, -1, 0, 0), (30, 40, 90, 10, 5, 30, 17, 3, 11), (20, 30, 60, 8, 8, 200, 25, 0, 4),
            (310, 1, 40, 3, 1, 5, 9, 0, 20), (1, 1500, 1500, 6, 2, 64, 100, 0, 6)]


@pytest.mark.parametrize("case", F32_ROWS, ids=lambda c: "-".join(map(str, c)))
def test_f32_rows(case):
    B, Tq, Tk, Hq, Hkv, D, left, right, sinks = case
    q, k, v = make(B, Tq, Tk, Hq, Hkv, D, "f32", gain=2.0)
    check(q, k, v, left, right, sinks)
    # lengths of their own; NaN and infinities behind the ends
    n = lens(*[Tq * (7 * i % (B + 1)) // B for i in range(B)])
    L = lens(*[x if Tq == Tk else max(x, Tk * (5 * i % (B + 1)) // B) for i, x in enumerate(n.tolist())])
    for b, x in enumerate(L.tolist()):
        k[b, x:], v[b, x:] = float("nan"), float("inf")
    check(q, k, v, left, right, sinks, q_len=n, kv_len=L)


def test_poison_in_many_rows():
    """as test_poison_beside_the_window, with the rows of many heads"""
    T, H = 400, 80
    q, k, v = make(1, T, T, 2 * H, H, 64, "f16")
    v[0, 150, :, 3] = float("inf")
    clean = v.clone()
    clean[0, 150, :, 3] = 0.0
    out = torch.empty_like(q)
    tpmd.attn_window(q, k, v, out, 10, 0, 0)
    tpmd.tpk_status()
    ref, bound, _ = reference(q, k, clean, 10, 0, 0, 64 ** -0.5)
    got = out.cpu().double()[0]
    bad = torch.zeros(T, 2 * H, 64, dtype=torch.bool)
    bad[150:161, :, 3] = True
    assert not bool(got[bad].isfinite().any())
    assert bool(((got - ref[0]).abs() <= bound[0])[~bad].all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_large_scores(dtype):
    """scores in the hundreds: the running maximum carries the softmax"""
    q, k, v = make(1, 300, 300, 2, 2, 64, dtype, gain=30.0)
    check(q, k, v, 100, 0, 4)
    check(q, k, v, 100, 0, 4, scale=-1.0)
    check(q, k, v, 100, 0, 4, scale=0.0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rising_scores(dtype):
    """every later key raises the maximum, and the other way round"""
    T, D = 700, 64
    q = torch.ones(1, T, 1, D)
    for sign in (1.0, -1.0):
        k = (torch.arange(T).float() * sign / 40)[None, :, None, None].expand(1, T, 1, D).contiguous()
        v = torch.randn(1, T, 1, D, generator=torch.Generator().manual_seed(1))
        check(*(t.to(TYPES[dtype]).cuda() for t in (q, k, v)), -1, -1, 0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_padded_batch_of_prompts(dtype):
    """sequences of their own lengths, one empty, one of a single token; what
    lies behind an end is NaN and is not looked at"""
    n = lens(260, 0, 1, 129, 259)
    q, k, v = make(5, 260, 260, 4, 2, 64, dtype)
    for b, x in enumerate(n.tolist()):
        for t in (q, k, v):
            t[b, x:] = float("nan")
    check(q, k, v, 50, 0, 3, q_len=n, kv_len=n)
    check(q, k, v, -1, 0, 0, q_len=n, kv_len=n)
    check(q, k, v, 20, 20, 1, q_len=n, kv_len=n)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("Tq", [1, 3])
def test_decode_over_stale_caches(dtype, Tq):
    """new tokens over caches of their own lengths; NaN and infinities
    everywhere that no row sees: behind the end and before the window"""
    L = [1500, Tq, 777, 128, 129, 1]
    q, k, v = make(6, Tq, 1500, 8, 2, 128, dtype)
    for b, x in enumerate(L):
        for t, bad in ((k, float("nan")), (v, float("inf"))):
            t[b, x:] = bad
            t[b, 4:max(4, x - Tq - 200)] = bad
    check(q, k, v, 200, 0, 4, kv_len=lens(*L))
    check(q, k, v, 200, 0, 4, kv_len=lens(*L), q_len=lens(Tq, 0, 1, Tq, Tq, 1))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows_that_see_nothing(dtype):
    """no keys at all; windows that end before the first key; lengths
    outside their range are clamped"""
    q, k, v = make(3, 4, 8, 2, 2, 64, dtype)
    check(q, k, v, 3, 0, 0, kv_len=lens(0, 2, 8))
    check(q, k, v, 3, 0, 2, kv_len=lens(-5, 1, 100), q_len=lens(4, 9, -1))
    check(q, k[:, :0], v[:, :0], -1, -1, 0)
    check(q, k[:, :0], v[:, :0], 3, 0, 2)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_poison_beside_the_window(dtype):
    """a NaN and an infinite value that only some rows see: the others keep
    their finite results"""
    T = 300
    q, k, v = make(1, T, T, 2, 1, 64, dtype)
    v[0, 150, 0, 3] = float("inf")
    v[0, 200, 0, 5] = float("nan")
    k[0, 250] = float("nan")
    out = torch.empty_like(q)
    tpmd.attn_window(q, k, v, out, 10, 0, 0)
    tpmd.tpk_status()
    clean_k, clean_v = k.clone(), v.clone()
    clean_v[0, 150, 0, 3] = clean_v[0, 200, 0, 5] = 0.0
    clean_k[0, 250] = 0.0
    ref, bound, _ = reference(q, clean_k, clean_v, 10, 0, 0, 64 ** -0.5)
    got = out.cpu().double()[0]
    t = torch.arange(T)
    bad = torch.zeros(T, 2, 64, dtype=torch.bool)
    bad[(t >= 150) & (t <= 160), :, 3] = True
    bad[(t >= 200) & (t <= 210), :, 5] = True
    bad[(t >= 250) & (t <= 260)] = True
    assert not bool(got[bad].isfinite().any())
    assert bool(((got - ref[0]).abs() <= bound[0])[~bad].all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_layouts(dtype):
    """packed q | k | v rows, heads before tokens, a cache that every
    sequence shares, rows that start off 16-byte boundaries, tokens in
    reverse order"""
    B, T, H, D = 2, 150, 4, 64
    g = torch.Generator().manual_seed(1)
    t = TYPES[dtype]
    packed = torch.randn(B, T, 3, H, D, generator=g).to(t).cuda()
    q, k, v = packed.unbind(2)
    a = check(q, k, v, 30, 4, 2)
    heads = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(a, check(*heads, 30, 4, 2, out=torch.empty(B, H, T, D, dtype=t, device="cuda").transpose(1, 2)))
    check(q, k[:1].expand(B, T, H, D), v[:1].expand(B, T, H, D), 30, 4, 2)
    check(q, k[:, :, :1].expand(B, T, H, D), v[:, :, :1].expand(B, T, H, D), 30, 0, 2)
    odd = torch.randn(B, T, 3, H, D + 3, generator=g).to(t).cuda()
    check(*odd[..., 1:D + 1].unbind(2), 30, 4, 2)
    wide = torch.full((B, T, H, D + 1), 5.0, dtype=t, device="cuda")
    check(q, k, v, 30, 4, 2, out=wide[..., 1:])
    assert bool((wide[..., 0] == 5.0).all())


def test_strided_view_with_a_wide_row():
    """few of the heads and columns of a wider buffer: the rest is not
    touched"""
    q, k, v = make(2, 200, 200, 8, 8, 128, "f16")
    big = torch.full((2, 200, 8, 128), 9.0, dtype=torch.float16, device="cuda")
    check(q[:, :, 2:5, 32:96], k[:, :, 2:5, 32:96], v[:, :, 2:5, 64:128], 60, 0, 1, out=big[:, :, 2:5, 32:96])
    keep = torch.ones_like(big, dtype=torch.bool)
    keep[:, :, 2:5, 32:96] = False
    assert bool((big[keep] == 9.0).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_offsets_past_32_bits(dtype):
    """tokens of a cache 2^26 elements apart: offsets beyond 2^31 elements"""
    T, D, step = 40, 64, 1 << 26
    buf = torch.empty(step * (T - 1) + 2 * D, dtype=TYPES[dtype], device="cuda")
    k = buf.as_strided((1, T, 1, D), (0, step, D, 1))
    v = buf.as_strided((1, T, 1, D), (0, step, D, 1), D)
    q, k0, v0 = make(1, T, T, 2, 1, D, dtype)
    k.copy_(k0)
    v.copy_(v0)
    check(q, k, v, 10, 0, 1)
    check(q[:, :1], k, v, -1, 0, 1)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_repeats_streams_and_graphs(dtype):
    """the same bits on every call, on two streams at once, and from a graph
    replayed on new inputs and lengths"""
    ins = [make(2, 1, 3000, 8, 2, 128, dtype, seed=s) for s in range(2)] + [make(1, 500, 500, 4, 2, 64, dtype)]
    want = [check(*x, 1000, 0, 4) for x in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    outs = [[torch.empty_like(w) for _ in range(6)] for w in want]
    torch.cuda.synchronize()
    for r in range(6):
        for i, x in enumerate(ins):
            tpmd.attn_window(*x, outs[i][r], 1000, 0, 4, stream=streams[i].cuda_stream)
    for i, st in enumerate(streams):
        tpmd.tpk_status(st.cuda_stream)
        assert all(torch.equal(o, want[i]) for o in outs[i])
    q, k, v = (x.clone() for x in ins[0])
    n = lens(3000, 3000)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tpmd.attn_window(q, k, v, out, 1000, 0, 4, kv_len=n, stream=torch.cuda.current_stream().cuda_stream)
    for L in ((3000, 1), (17, 2999), (0, 500)):
        n.copy_(torch.tensor(L, dtype=torch.int32))
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, check(q, k, v, 1000, 0, 4, kv_len=n))


def test_decode_continues_a_prompt():
    """the rows of a prompt, and the same rows one new token at a time over
    the growing cache, agree within both bounds"""
    T = 40
    q, k, v = make(2, T, T, 4, 2, 64, "f16")
    whole = check(q, k, v, 12, 0, 3)
    ref, bound, _ = reference(q, k, v, 12, 0, 3, 0.125)
    for t in range(T):
        one = torch.empty_like(q[:, :1])
        tpmd.attn_window(q[:, t:t + 1], k, v, one, 12, 0, 3, kv_len=lens(t + 1, t + 1))
        assert bool(((one[:, 0].cpu().double() - whole[:, t].cpu().double()).abs() <= 2 * bound[:, t]).all())


def test_block_of_the_sampler():
    """quantise -> q | k | v product -> attention -> quantise -> output
    product, as a transformer block runs them, against float64 from each
    step's own inputs"""
    F8 = torch.float8_e4m3fn
    g = torch.Generator().manual_seed(6)
    B, T, H, nh = 3, 60, 256, 2
    x = torch.randn(B * T, H, generator=g).cuda()
    wqkv, wo = (torch.randn(n, H, generator=g).cuda() / 16 for n in (3 * H, H))

    def quant(t, rows):
        q = torch.empty(t.shape, dtype=F8, device="cuda")
        s = torch.empty(-(-t.shape[0] // rows), -(-t.shape[1] // 128), device="cuda")
        return tpmd.quant_f8(t, q, s, rows=rows)

    def real(q, s, rows):
        s = s.cpu().double().repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]
        return q.cpu().double() * s

    xq, wq, wp = quant(x, 1), quant(wqkv, 128), quant(wo, 128)
    qkv = torch.empty(B * T, 3 * H, dtype=torch.float16, device="cuda")
    tpmd.gemm_f8(*xq, *wq, qkv)
    q, k, v = qkv.view(B, T, 3, nh, H // nh).unbind(2)
    att = check(q, k, v, 2, 2, 10)
    aq = quant(att.view(B * T, H), 1)
    y = torch.empty(B * T, H, device="cuda")
    tpmd.gemm_f8(*aq, *wp, y)
    tpmd.tpk_status()
    a, b = real(*xq, 1), real(*wq, 128)
    err = (qkv.cpu().double() - a @ b.t()).abs()
    assert bool((err <= (128 + 8) * 2.0 ** -23 * (a.abs() @ b.abs().t()) + 2.0 ** -11 * (a @ b.t()).abs() + 2.0 ** -25).all())
    a, b = real(*aq, 1), real(*wp, 128)
    err = (y.cpu().double() - a @ b.t()).abs()
    assert bool((err <= (128 + 8) * 2.0 ** -23 * (a.abs() @ b.abs().t())).all())
