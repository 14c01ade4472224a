"""Refusals of the 8-bit and windowed-attention op entry points: every bad
argument is an error on the host, before anything reaches a GPU (needs none;
the pointers are host addresses that no accepted call would read)."""
from __future__ import annotations

import ctypes as C
import struct

import pytest
import torch

import tpmd

BUF = C.create_string_buffer(4096)
P = (C.addressof(BUF) + 255) & ~255


def _err():
    return tpmd.load_library().tpk_last_error().decode()


def _quant(**kw):
    a = dict(x=P, dtype=0, ldx=128, M=4, K=128, rows=1, q=P, ldq=128, s=P, lds=1)
    a.update(kw)
    return tpmd.load_library().tpk_quant_f8(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=2), "dtype"), (dict(dtype=7), "dtype"), (dict(rows=64), "rows"), (dict(rows=0), "rows"),
    (dict(M=-1), "shape"), (dict(K=-1), "shape"), (dict(x=None), "null"), (dict(q=None), "null"),
    (dict(s=None), "null"), (dict(ldq=127), "row stride"), (dict(ldx=-128), "row stride"),
    (dict(K=256, ldx=256, ldq=256, lds=1), "row stride"), (dict(x=P + 2), "element type"), (dict(s=P + 1), "element type")])
def test_quant_refuses(kw, msg):
    assert _quant(**kw) == -1 and msg in _err()


def _gemm(**kw):
    a = dict(X=P, ldx=128, sx=P, ldsx=1, W=P, ldw=128, sw=P, ldsw=1, Y=P, ldy=64, yd=0, sy=None, ldsy=0, M=4, N=64,
             K=128, bias=None, act=0)
    a.update(kw)
    return tpmd.load_library().tpk_gemm_f8(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(yd=3), "y_dtype"), (dict(act=4), "act"), (dict(act=-1), "act"), (dict(M=-1), "shape"), (dict(K=0), "shape"),
    (dict(K=-5), "shape"), (dict(M=(1 << 30) + 1), "shape"), (dict(N=(1 << 30) + 1, ldy=1 << 31), "shape"), (dict(yd=2), "sy goes"), (dict(sy=P), "sy goes"), (dict(X=None), "null"),
    (dict(W=None), "null"), (dict(sx=None), "null"), (dict(sw=None), "null"), (dict(Y=None), "null"),
    (dict(X=P + 8), "16-byte"), (dict(W=P + 1), "16-byte"), (dict(ldx=136), "16-byte"), (dict(ldw=129), "16-byte"),
    (dict(ldx=112), "row stride"), (dict(ldy=63), "row stride"), (dict(K=256, ldx=256, ldw=256), "row stride"),
    (dict(N=200, ldy=200, ldsw=0), "row stride"), (dict(sx=P + 2), "element type"), (dict(Y=P + 1), "element type"),
    (dict(bias=P + 1), "element type"), (dict(yd=2, sy=P, ldsy=0), "row stride")])
def test_gemm_refuses(kw, msg):
    assert _gemm(**kw) == -1 and msg in _err()


def _attn(**kw):
    a = dict(q=P, k=P, v=P, out=P, strides=(512, 128, 64) * 4, dtype=1, B=1, Tq=4, Tk=4, Hq=2, Hkv=2, D=64, ql=None,
             kl=None, left=1, right=0, sinks=0, scale=0.125)
    a.update(kw)
    if a["strides"] is not None:
        a["strides"] = (C.c_int64 * 12)(*a["strides"])
    return tpmd.load_library().tpk_attn_window(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=2), "dtype"), (dict(B=-1), "shape"), (dict(Tq=-1), "shape"), (dict(Tk=(1 << 30) + 1), "shape"),
    (dict(D=0), "shape"), (dict(D=257), "shape"), (dict(Hkv=3), "multiple"), (dict(Hkv=0), "multiple"),
    (dict(sinks=-1), "sinks"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(out=None), "null"),
    (dict(strides=None), "null"), (dict(q=P + 1), "element type"), (dict(kl=P + 2), "element type"),
    (dict(strides=(512, 128, 64) * 3 + (512, 64, 64)), "overlap"),
    (dict(strides=(512, 128, 64) * 3 + (512, 128, 63)), "overlap"),
    (dict(B=2, strides=(512, 128, 64) * 3 + (0, 128, 64)), "overlap"),
    (dict(B=2, strides=(512, 128, 64) * 3 + (500, 128, 64)), "overlap")])
def test_attn_refuses(kw, msg):
    assert _attn(**kw) == -1 and msg in _err()


def test_nothing_to_do():
    """no rows: success, pointers not looked at"""
    assert _quant(M=0, x=None, q=None, s=None) == 0 and _quant(K=0, x=None, q=None, s=None) == 0
    assert _gemm(M=0, X=None, Y=None) == 0 and _gemm(N=0, W=None, Y=None) == 0
    assert _attn(B=0, q=None, out=None) == 0 and _attn(Tq=0, q=None) == 0 and _attn(Hq=0, Hkv=0, q=None) == 0


def test_host_memory_is_refused():
    """an accepted shape with host pointers: refused (here: no device, or
    memory that is not the device's)"""
    for call in (_quant, _gemm, _attn):
        assert call() == -1
        assert "device" in _err()


def test_binding_refuses():
    """the Python checks, on CPU tensors (refused before the library is called)"""
    f8 = torch.float8_e4m3fn
    x, q, s = torch.zeros(4, 200), torch.zeros(4, 200, dtype=f8), torch.zeros(4, 2)
    for bad in (dict(rows=2), dict(x=x.double()), dict(q=q[:, :100]), dict(s=s[:2]), dict(s=s.half()),
                dict(q=torch.zeros(200, 4, dtype=f8).t())):
        with pytest.raises(tpmd.TpmdError):
            tpmd.quant_f8(**{**dict(x=x, q=q, s=s), **bad})
    w, sw, y = torch.zeros(130, 200, dtype=f8), torch.zeros(2, 2), torch.zeros(4, 130)
    for bad in (dict(X=x), dict(sx=s[:, :1]), dict(W=w[:, :100]), dict(sw=s), dict(Y=y[:, :1]), dict(Y=y.to(f8)),
                dict(sy=s), dict(bias=torch.zeros(4)), dict(Y=y.double()), dict(Y=y.to(f8), sy=s[:, :1])):
        with pytest.raises(tpmd.TpmdError):
            tpmd.gemm_f8(**{**dict(X=q, sx=s, W=w, sw=sw, Y=y), **bad})
    a = dict(q=torch.zeros(2, 3, 4, 8), k=torch.zeros(2, 5, 2, 8), v=torch.zeros(2, 5, 2, 8), out=torch.zeros(2, 3, 4, 8),
             left=1)
    for bad in (dict(q=a["q"].half()), dict(k=a["k"][:1]), dict(v=a["v"][:, :4]), dict(out=a["out"][:, :2]),
                dict(q_len=torch.zeros(2)), dict(kv_len=torch.zeros(3, dtype=torch.int32)),
                dict(q=torch.zeros(2, 3, 8, 4).transpose(2, 3))):
        with pytest.raises(tpmd.TpmdError):
            tpmd.attn_window(**{**a, **bad})


def _words(args):
    """Arguments as a packed call takes them: 8 bytes each, strides in their place"""
    w = []
    for a in args:
        if isinstance(a, float):
            w.append(struct.pack("d", a))
        else:
            w += [struct.pack("q", x or 0) for x in (a if isinstance(a, tuple) else (a,))]
    return b"".join(w)


@pytest.mark.parametrize("name,args,msg", [
    ("quant_f8", (P, 0, 128, 4, 128, 64, P, 128, P, 1, None), "rows"),
    ("quant_f8", (P, 0, 128, 4, 128, 1, P, 128, P + 1, 1, None), "element type"),
    ("quant_f8", (P, 0, 128, 4, 128, 1, P, 127, P, 1, None), "row stride"),
    ("quant_f8", (P, 0, 128, 4, 128, 1 << 32 | 1, P, 128, P, 1, None), "range"),
    ("gemm_f8", (P, 128, P, 1, P, 128, P, 1, P, 64, 0, None, 0, 4, 64, 128, None, 4, None), "act"),
    ("gemm_f8", (P, 128, P, 1, P, 128, P, 1, P, 64, 0, None, 0, 4, 64, 128, P + 1, 0, None), "element type"),
    ("gemm_f8", (P, 128, P, 1, P, 128, P, 1, P, 64, 0, None, 0, 1 << 32 | 4, 64, 128, None, 0, None), "range"),
    ("attn_window", (P, P, P, P, (512, 128, 64) * 4, 1, 1, 4, 4, 2, 2, 64, None, P + 1, 1, 0, 0, 0.125, None), "element type"),
    ("attn_window", (P, P, P, P, (512, 128, 64) * 4, 1, 1, 4, 4, 2, 2, 64, None, None, 1, 0, -1, 0.125, None), "sinks"),
    ("attn_window", (P, P, P, P, (512, 128, 64) * 4, 1, 1, 4, 4, 2, 2, 64, None, None, 1, 0, 0, float("inf"), None), "scale"),
    ("attn_window", (P, P, P, P, (512, 128, 64) * 3 + (512, 64, 64), 1, 1, 4, 4, 2, 2, 64, None, None, 1, 0, 0, 0.125, None), "overlap"),
    ("attn_window", (P, P, P, P, (512, 128, 64) * 4, 1, 1, 4, 4, 2, 2, 64, None, None, 1 << 31, 0, 0, 0.125, None), "range")])
def test_packed_calls_refuse_alike(name, args, msg):
    """Each word reaches the argument of its place: the last ones of a kind are the bad ones here"""
    assert getattr(tpmd.load_library(), f"tpk_{name}_packed")(_words(args)) == -1
    assert msg in _err() and f"tpk_{name}:" in _err()
