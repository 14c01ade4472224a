"""Timing cases of the operators around the sampler's transformer block: quantisation to 8-bit floating point
(tpmd.quant_f8), the matrix product with a scale per block of 128 (tpmd.gemm_f8), and attention over a sliding
window with first tokens that stay visible (tpmd.attn_window).

With `own` false, run() computes each operator in its plain form from elementary torch operations in float32; with
`own` true it makes the calls a user makes of the library. exact() evaluates the definitions in float64."""
import math
import os
import sys

import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0      # largest e4m3 value
S_MIN = 2.0 ** -126  # smallest scale (a block of zeros)
TYPES = {"f16": torch.float16, "f32": torch.float32, "f8": F8}
ACTS = {"none": 0, "gelu": 1, "gelu_tanh": 2}
DEV = "cuda"


def _cdiv(a, b):
    return -(-a // b)


def listed():
    return [
        # the sampler's block input: 3 guidance branches x 60 frames, width 1024, on its way into a linear
        dict(name="quant_sampler_rows", op="quant", m=180, k=1024, dtype="f32", rows=1),
        # one MLP weight of the sampler, quantised when the weights are prepared
        dict(name="quant_weight_blocks", op="quant", m=4096, k=1024, dtype="f32", rows=128),
        # the rows of many clips batched together, f16 activations
        dict(name="quant_many_rows", op="quant", m=16384, k=4096, dtype="f16", rows=1),
        # the sampler's first MLP linear: bias, tanh GELU, its output quantised for the second one
        dict(name="gemm_fc1_gelu_f8", op="gemm", m=180, n=4096, k=1024, out="f8", act="gelu_tanh", bias=True),
        # the sampler's second MLP linear: a long sum for few outputs
        dict(name="gemm_fc2", op="gemm", m=180, n=1024, k=4096, out="f32", act="none", bias=True),
        # odd sizes everywhere: rows, columns and a last k block of 16
        dict(name="gemm_odd", op="gemm", m=777, n=1000, k=528, out="f16", act="gelu", bias=True),
        # many clips at once: compute bound
        dict(name="gemm_many_rows", op="gemm", m=8192, n=4096, k=4096, out="f16", act="none", bias=False),
        # the sampler's attention: 60 frames, a band of five, the 10 context frames visible throughout
        dict(name="attn_sampler_f32", op="attn", dtype="f32", b=3, tq=60, tk=60, hq=8, hkv=8, d=128, left=2, right=2,
             sinks=10, ragged=False),
        # streaming: one new token a sequence over a cache, sequences of different lengths
        dict(name="attn_decode", op="attn", dtype="f16", b=16, tq=1, tk=8192, hq=16, hkv=4, d=128, left=4095, right=0,
             sinks=4, ragged=True),
        # five minutes of audio frames at 25 per second, five seconds to either side
        dict(name="attn_long_audio", op="attn", dtype="f16", b=1, tq=7500, tk=7500, hq=12, hkv=12, d=64, left=125,
             right=125, sinks=0, ragged=False),
        # a padded batch of odd lengths (one of them empty) and an odd head width
        dict(name="attn_padded_batch", op="attn", dtype="f16", b=5, tq=1111, tk=1111, hq=6, hkv=2, d=80, left=255,
             right=0, sinks=3, ragged=True),
        # a long causal prompt with a wide window: compute bound
        dict(name="attn_long_prompt", op="attn", dtype="f16", b=1, tq=16384, tk=16384, hq=16, hkv=4, d=128, left=4095,
             right=0, sinks=4, ragged=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: any operator, sizes over the listed range (log-uniform), odd ones among them."""
    op = rng.choice(["quant", "gemm", "gemm", "attn", "attn", "attn"])
    if op == "quant":
        return dict(op=op, m=_log_int(rng, 1, 16384), k=_log_int(rng, 8, 4096), dtype=rng.choice(["f16", "f32"]),
                    rows=rng.choice([1, 1, 128]))
    if op == "gemm":
        while True:
            c = dict(op=op, m=_log_int(rng, 1, 8192), n=_log_int(rng, 16, 8192), k=_log_int(rng, 32, 8192),
                     out=rng.choice(["f32", "f16", "f8"]), act=rng.choice(["none", "gelu", "gelu_tanh"]),
                     bias=rng.choice([True, False]))
            if c["m"] * c["n"] * c["k"] <= 8192 * 4096 * 4096:
                return c
    while True:
        hkv = rng.choice([1, 2, 3, 4, 8, 12])
        c = dict(op=op, dtype=rng.choice(["f16", "f16", "f16", "f32"]), hkv=hkv, hq=hkv * rng.choice([1, 1, 2, 3, 4, 8]),
                 d=rng.choice([32, 40, 64, 64, 80, 96, 128, 128]), sinks=rng.choice([0, 1, 4, 10, 130]),
                 ragged=rng.choice([True, False]))
        kind = rng.choice(["decode", "prefill", "prefill", "band"])
        c["left"] = _log_int(rng, 1, 4096) - 1 if rng.random() < 0.85 else -1
        if kind == "decode":  # few new tokens over a cache
            c.update(b=_log_int(rng, 1, 64), tq=rng.choice([1, 1, 1, 2, 5]), tk=_log_int(rng, 8, 16384), right=0)
            c["tq"] = min(c["tq"], c["tk"])
        elif kind == "prefill":
            t = _log_int(rng, 1, 16384)
            c.update(b=rng.choice([1, 1, 2, 5]), tq=t, tk=t, right=0)
        else:  # to either side
            t = _log_int(rng, 1, 16384)
            c.update(b=rng.choice([1, 1, 3]), tq=t, tk=t, right=rng.choice([c["left"], 7]))
        cost = _attn_pairs(c) * c["hq"] * c["d"] * 4
        most = _attn_pairs(listed()[-1]) * 16 * 128 * 4
        # the float32 form is the parity path: sizes of one clip
        if cost <= (most if c["dtype"] == "f16" else most / 32) and c["b"] * c["tk"] * c["hkv"] * c["d"] <= 1 << 27:
            return c


def _lens(c):
    """(new tokens, cache length) of each sequence: part of the case, as a scheduler's plan is."""
    if not c["ragged"]:
        return [(c["tq"], c["tk"])] * c["b"]
    got = []
    for i in range(c["b"]):
        if c["tq"] == c["tk"]:  # a padded batch of prompts: the first full, the last empty if there are several
            n = c["tq"] * (c["b"] - 1 - i) // max(1, c["b"] - 1) if c["b"] > 1 else _cdiv(2 * c["tq"], 3)
            got.append((n, n))
        else:  # a cache filled to half at least
            got.append((c["tq"], max(c["tq"], c["tk"] - (c["tk"] // 2) * i // c["b"])))
    return got


def _attn_pairs(c):
    """Visible (query, key) pairs of all sequences."""
    total = 0
    for n, length in _lens(c):
        if n <= 0:
            continue
        pos = torch.arange(length - n, length, dtype=torch.int64)
        hi = torch.clamp(pos + c["right"] + 1, max=length) if c["right"] >= 0 else torch.full_like(pos, length)
        lo = torch.clamp(pos - c["left"], min=0) if c["left"] >= 0 else torch.zeros_like(pos)
        first = torch.minimum(torch.minimum(torch.full_like(pos, c["sinks"]), lo), hi)
        total += int((hi - lo).clamp(min=0).sum() + first.clamp(min=0).sum())
    return total


def work(case):
    c = case
    if c["op"] == "quant":
        es = 2 if c["dtype"] == "f16" else 4
        return {"bytes": c["m"] * c["k"] * (es + 1) + 4 * _cdiv(c["m"], c["rows"]) * _cdiv(c["k"], 128),
                "flops": 3 * c["m"] * c["k"]}
    if c["op"] == "gemm":
        m, n, k, kb = c["m"], c["n"], c["k"], _cdiv(c["k"], 128)
        out = m * n * {"f32": 4, "f16": 2, "f8": 1}[c["out"]] + (4 * m * _cdiv(n, 128) if c["out"] == "f8" else 0)
        return {"bytes": (m + n) * k + 4 * kb * (m + _cdiv(n, 128)) + (4 * n if c["bias"] else 0) + out,
                "flops": 2 * m * n * k}
    es = 2 if c["dtype"] == "f16" else 4
    rows = keys = 0
    for n, length in _lens(c):
        if n <= 0 or length <= 0:
            continue
        rows += n
        # the keys that some query of the sequence sees
        hi = min(length, length + c["right"]) if c["right"] >= 0 else length
        lo = max(0, length - n - c["left"]) if c["left"] >= 0 else 0
        keys += hi - lo + min(lo, c["sinks"])
    return {"bytes": es * c["d"] * (2 * rows * c["hq"] + 2 * keys * c["hkv"]),
            "flops": 4 * c["d"] * c["hq"] * _attn_pairs(c)}


# ---- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _activations(m, k, g):
    """Rows as a normalised, modulated block input has them: some channels several times larger than others."""
    gain = torch.exp(0.7 * torch.randn(k, generator=g, device=DEV))
    return torch.randn(m, k, generator=g, device=DEV) * gain


def _padded(m, k, dtype, pad=16):
    """[m][k] with rows that start on 16-byte boundaries."""
    return torch.zeros(m, _cdiv(k, pad) * pad, dtype=dtype, device=DEV)[:, :k]


def _block_quant(x, rows):
    """(values / scale rounded to e4m3, scales): scale = max(amax / 448, 2^-126) of each block of rows x 128."""
    m, k = x.shape
    mb, kb = _cdiv(m, rows), _cdiv(k, 128)
    x = x.float()
    full = torch.zeros(mb * rows, kb * 128, dtype=torch.float32, device=x.device)
    full[:m, :k] = x
    blocks = full.view(mb, rows, kb, 128)
    amax = blocks.abs().amax(dim=3).amax(dim=1)
    # F8_MAX as a tensor: a division, not a product with the reciprocal
    s = torch.clamp(amax / torch.full_like(amax, F8_MAX), min=S_MIN)
    q = (blocks / s[:, None, :, None]).clamp(-F8_MAX, F8_MAX)
    return q.reshape(mb * rows, kb * 128)[:m, :k].to(F8), s


def prepare(case, seed):
    c, g = case, _gen(seed)
    st = {"case": c}
    if own:
        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        pkg = os.path.join(here, "talking-portrait.cpp_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import tpmd
        tpmd.load_library()
        st["tpmd"] = tpmd
    if c["op"] == "quant":
        x = _activations(c["m"], c["k"], g) if c["rows"] == 1 else \
            torch.randn(c["m"], c["k"], generator=g, device=DEV) / math.sqrt(c["k"])
        st["x"] = x.to(TYPES[c["dtype"]])
        st["q"] = _padded(c["m"], c["k"], F8)
        st["s"] = torch.zeros(_cdiv(c["m"], c["rows"]), _cdiv(c["k"], 128), device=DEV)
    elif c["op"] == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        for name, rows, v in (("x", 1, _activations(m, k, g)),
                              ("w", 128, torch.randn(n, k, generator=g, device=DEV) / math.sqrt(2.0 * k))):
            q, s = _block_quant(v, rows)
            st[name], st["s" + name] = _padded(q.shape[0], k, F8), s
            st[name].copy_(q)
        st["bias"] = 0.3 * torch.randn(n, generator=g, device=DEV) if c["bias"] else None
        st["y"] = _padded(m, n, TYPES[c["out"]])
        st["sy"] = torch.zeros(m, _cdiv(n, 128), device=DEV) if c["out"] == "f8" else None
    else:
        t = TYPES[c["dtype"]]
        # one buffer of cache rows [B][T][Hkv][D] each for k and v; places behind a sequence's end hold old values
        for name, length, heads in (("q", c["tq"], c["hq"]), ("k", c["tk"], c["hkv"]), ("v", c["tk"], c["hkv"])):
            st[name] = torch.randn(c["b"], length, heads, c["d"], generator=g, device=DEV).to(t)
        st["out"] = torch.zeros(c["b"], c["tq"], c["hq"], c["d"], dtype=t, device=DEV)
        st["lens"] = _lens(c)
        st["q_len"] = st["kv_len"] = None
        if c["ragged"]:
            st["q_len"] = torch.tensor([n for n, _ in st["lens"]], dtype=torch.int32, device=DEV)
            st["kv_len"] = torch.tensor([n for _, n in st["lens"]], dtype=torch.int32, device=DEV)
    return st


# ---- plain forms

def _act(v, act):
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_gemm(st):
    c = st["case"]
    m, n, k = c["m"], c["n"], c["k"]
    x = st["x"].float() * st["sx"].repeat_interleave(128, dim=1)[:, :k]
    w = st["w"].float() * st["sw"].repeat_interleave(128, dim=0)[:n].repeat_interleave(128, dim=1)[:, :k]
    y = x @ w.t()
    if st["bias"] is not None:
        y = y + st["bias"]
    y = _act(y, c["act"])
    if c["out"] == "f8":
        q, s = _block_quant(y, 1)
        return {"y": q, "sy": s}
    return {"y": y.to(TYPES[c["out"]])}


def _visible(c, pos, key, length):
    """Whether the queries at positions `pos` see the keys `key` (both int64, broadcast together)."""
    ok = key < length
    if c["right"] >= 0:
        ok = ok & (key <= pos + c["right"])
    near = key < c["sinks"]
    near = near | (key >= pos - c["left"]) if c["left"] >= 0 else torch.ones_like(ok)
    return ok & near


def _plain_rows(c, q, k, v, ok):
    """q [..., n, g, D] in groups of g query heads, k and v [..., j, D], ok [..., n, j] -> [..., n, g, D]"""
    n, g = q.shape[-3], q.shape[-2]
    s = q.flatten(-3, -2) @ k.transpose(-1, -2) * (1.0 / math.sqrt(c["d"]))
    s = s.unflatten(-2, (n, g))
    ok = ok[..., :, None, :]
    s = torch.where(ok, s, torch.full_like(s, -math.inf))
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    o = (p.flatten(-3, -2) @ v).unflatten(-2, (n, g))
    return torch.where(total > 0, o / total, torch.zeros_like(o))


def _plain_attn(st):
    c = st["case"]
    b, tq, tk, hq, hkv, d = c["b"], c["tq"], c["tk"], c["hq"], c["hkv"], c["d"]
    g = hq // hkv
    out = torch.zeros(b, tq, hq, d, dtype=TYPES[c["dtype"]], device=DEV)
    if b * tq * tk * hq <= 1 << 28:  # every sequence at once
        nq = torch.tensor([n for n, _ in st["lens"]], device=DEV)[:, None, None]
        nk = torch.tensor([n for _, n in st["lens"]], device=DEV)[:, None, None]
        row = torch.arange(tq, device=DEV)[None, :, None]
        ok = _visible(c, row + nk - nq, torch.arange(tk, device=DEV)[None, None, :], nk)
        q = st["q"].float().view(b, tq, hkv, g, d).permute(0, 2, 1, 3, 4)
        k, v = (st[x].float().permute(0, 2, 1, 3) for x in "kv")
        o = _plain_rows(c, q, k, v, ok[:, None]).permute(0, 2, 1, 3, 4).reshape(b, tq, hq, d)
        return torch.where((row < nq)[..., None], o.to(out.dtype), out)
    for i, (n, length) in enumerate(st["lens"]):  # 512 queries at a time, with the keys that they see
        for r0 in range(0, n, 512):
            r1 = min(n, r0 + 512)
            p0, p1 = length - n + r0, length - n + r1 - 1
            hi = min(length, p1 + c["right"] + 1) if c["right"] >= 0 else length
            lo = max(0, p0 - c["left"]) if c["left"] >= 0 else 0
            key = torch.arange(lo, hi, device=DEV)
            if min(c["sinks"], lo):
                key = torch.cat([torch.arange(min(c["sinks"], lo), device=DEV), key])
            pos = torch.arange(p0, p1 + 1, device=DEV)
            ok = _visible(c, pos[:, None], key[None, :], length)
            q = st["q"][i, r0:r1].float().view(r1 - r0, hkv, g, d).transpose(0, 1)
            k, v = (st[x][i].index_select(0, key).float().transpose(0, 1) for x in "kv")
            o = _plain_rows(c, q, k, v, ok[None])
            out[i, r0:r1] = o.transpose(0, 1).reshape(r1 - r0, hq, d).to(out.dtype)
    return out


def run(state):
    st, c = state, state["case"]
    if c["op"] == "quant":
        if own:
            st["tpmd"].quant_f8(st["x"], st["q"], st["s"], rows=c["rows"])
            return {"q": st["q"], "s": st["s"]}
        q, s = _block_quant(st["x"], c["rows"])
        return {"q": q, "s": s}
    if c["op"] == "gemm":
        if own:
            st["tpmd"].gemm_f8(st["x"], st["sx"], st["w"], st["sw"], st["y"], sy=st["sy"], bias=st["bias"],
                               act=ACTS[c["act"]])
            return {"y": st["y"], "sy": st["sy"]} if c["out"] == "f8" else {"y": st["y"]}
        return _plain_gemm(st)
    if own:
        st["tpmd"].attn_window(st["q"], st["k"], st["v"], st["out"], left=c["left"], right=c["right"],
                               sinks=c["sinks"], q_len=st["q_len"], kv_len=st["kv_len"])
        return st["out"]
    return _plain_attn(st)


# ---- the definitions in float64

def _exact_f8(v):
    """float64 values rounded to the nearest e4m3 value, ties to even, saturating at 448."""
    a = v.abs().clamp(max=F8_MAX)
    _, e = torch.frexp(a)                       # a = f 2^e, f in [1/2, 1)
    step = torch.ldexp(torch.ones_like(a), torch.clamp(e - 1, min=-6) - 3)
    return torch.sign(v) * torch.round(a / step) * step


def _exact_quant(x, rows):
    m, k = x.shape
    q, s = torch.empty_like(x), torch.empty(_cdiv(m, rows), _cdiv(k, 128), dtype=x.dtype, device=x.device)
    for j in range(s.shape[1]):
        cols = x[:, 128 * j:128 * j + 128]
        top = cols.abs().amax(dim=1)
        if rows > 1:
            top = torch.nn.functional.pad(top, (0, s.shape[0] * rows - m)).view(-1, rows).amax(dim=1)
        s[:, j] = torch.clamp(top / F8_MAX, min=S_MIN)
        q[:, 128 * j:128 * j + 128] = _exact_f8(cols / s[:, j].repeat_interleave(rows)[:m, None])
    return q, s


def exact(case, seed):
    c = case
    st = prepare(c, seed)
    if c["op"] == "quant":
        q, s = _exact_quant(st["x"].double(), c["rows"])
        return {"q": q, "s": s}
    if c["op"] == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        y = torch.zeros(m, n, dtype=torch.float64, device=DEV)
        for j in range(_cdiv(k, 128)):  # a block of 128 at a time, its scales on its sums
            cols = slice(128 * j, min(k, 128 * j + 128))
            part = st["x"][:, cols].double() @ st["w"][:, cols].double().t()
            y += part * st["sx"][:, j].double()[:, None] * st["sw"][:, j].double().repeat_interleave(128)[None, :n]
        if st["bias"] is not None:
            y += st["bias"].double()
        if c["act"] == "gelu":
            y = y * 0.5 * torch.special.erfc(-y / math.sqrt(2.0))
        elif c["act"] == "gelu_tanh":
            y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
        if c["out"] == "f8":
            q, s = _exact_quant(y, 1)
            return {"y": q, "sy": s}
        return {"y": y}
    out = torch.zeros(c["b"], c["tq"], c["hq"], c["d"], dtype=torch.float64, device=DEV)
    for i, (n, length) in enumerate(st["lens"]):
        for h in range(c["hq"]):
            k, v = (st[x][i, :length, h // (c["hq"] // c["hkv"])].double() for x in "kv")
            for r0 in range(0, n, 1024):
                pos = torch.arange(r0, min(n, r0 + 1024), device=DEV) + (length - n)
                first = max(0, int(pos[0]) - c["left"]) if c["left"] >= 0 else 0
                last = min(length, int(pos[-1]) + c["right"] + 1) if c["right"] >= 0 else length
                key = torch.arange(length, device=DEV)
                key = key[(key < c["sinks"]) & (key < first) | (key >= first) & (key < last)]
                away = torch.zeros(len(pos), len(key), dtype=torch.bool, device=DEV)
                if c["left"] >= 0:
                    away |= (pos[:, None] - key[None, :] > c["left"]) & (key[None, :] >= c["sinks"])
                if c["right"] >= 0:
                    away |= key[None, :] - pos[:, None] > c["right"]
                s = (st["q"][i, r0:r0 + len(pos), h].double() @ k[key].t() / math.sqrt(c["d"])).masked_fill(away, -math.inf)
                out[i, r0:r0 + len(pos), h] = torch.nan_to_num(torch.softmax(s, dim=1)) @ v[key]
    return out
