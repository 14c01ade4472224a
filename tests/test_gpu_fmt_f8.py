"""The sampler with its qkv, MLP and adaLN linears in 8-bit floating point
(TPMD_DTYPE_F8), against the float64 torch DiT.

A quantised operand is off by at most 2^-4 of its value, 2^-4 / sqrt(3) =
0.036 rms; errors of either sign in both operands leave a product's sum off by
0.051 of its rms. The sub-blocks' errors add in squares along the residual
stream (norms do not amplify): 5 linears a block (the modulations count as
one) give 0.051 sqrt(5 depth + 1), and 1 - cosine is half its square: 0.015
at depth 2, 0.053 at depth 8.

The same DiT with the same operands quantised in float64 is no closer than
that has to be: an operand that differs by d relative (2^-11 from f16 at
first) crosses a border between e4m3 values 2^-4 apart with probability
16 d and is then off by a step, so operands of a linear are off by sqrt(d /
16) rms on its far side: 2^-11 makes 0.006, 0.006 makes 0.019, 0.019 makes
0.034, the error of an independent quantisation (0.036). From the second
linear in a row on, the two differ like two independent quantisations, with
the sum of both squares: 1 - cosine up to 0.051^2 (5 depth + 1), 0.029 at
depth 2 and 0.107 at depth 8. What it adds to the comparison with the
unquantised DiT is that both go the same way where a scale or a block were
wrong by a factor."""
import numpy as np
import pytest
import torch

import torch_lia
import tpmd
from metrics import cosine
from tpmd import synth

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _inputs(cfg, seed=1):
    rng = np.random.default_rng(seed)
    T = cfg["chunk_frames"] + cfg["prev_frames"]
    CD = cfg["dim_w"] + cfg["dim_a"] + cfg["dim_e"]
    return (rng.standard_normal((T, cfg["dim_w"])).astype(np.float32),
            rng.standard_normal((3, T, CD)).astype(np.float32))


def _quant(x, rows):
    """x rounded as tpk_quant_f8 rounds it, in float64"""
    shape = x.shape
    x = x.reshape(-1, shape[-1])
    M, K = x.shape
    mb, kb = -(-M // rows), -(-K // 128)
    full = torch.zeros(mb * rows, kb * 128, dtype=torch.float64)
    full[:M, :K] = x
    b = full.view(mb, rows, kb, 128)
    s = (b.abs().amax(dim=(1, 3), keepdim=True) / 448.0).clamp(min=2.0 ** -126)
    return ((b / s).float().clamp(-448, 448).to(F8).double() * s).view(mb * rows, kb * 128)[:M, :K].reshape(shape)


class QuantFmt(torch_lia.TorchFmt):
    """the DiT with the 8-bit linears' operands quantised"""

    def __init__(self, cfg, raw):
        super().__init__(cfg, raw)
        ada = [n for n in self.w if "adaLN_modulation" in n and n.endswith(".weight")]
        ada.sort(key=lambda n: int(n.split(".")[1]) if n.startswith("blocks.") else 1 << 30)
        both = _quant(torch.cat([self.w[n] for n in ada]), 128)  # one matrix, blocks of 128 rows across it
        at = 0
        for n in ada:
            rows = self.w[n].shape[0]
            self.w[n] = both[at:at + rows]
            at += rows
        for n in self.w:
            if n.endswith(".weight") and (".attn.qkv" in n or ".mlp." in n) and not n.startswith("t_embedder."):
                self.w[n] = _quant(self.w[n], 128)

    def _lin(self, n, x):
        if (".attn.qkv" in n or ".mlp." in n or "adaLN" in n) and not n.startswith("t_embedder."):
            x = _quant(x, 1)
        return super()._lin(n, x)


def _sampler(cfg, w, dtype=tpmd.DTYPE_F8):
    s = tpmd.FmtSampler(cfg, 0, dtype)
    s.set_tensors(w)
    s.prepare()
    return s


CASES = [(synth.FMT_SMALL, 0.985, 0.971), (dict(synth.FMT_SMALL, dim_h=208, n_heads=2, attn_window=9), 0.985, 0.971),
         (synth.FMT_CONFIG, 0.947, 0.893)]


@pytest.mark.parametrize("cfg,gate,gate_q", CASES, ids=["small", "odd", "config4"])
def test_forward(cfg, gate, gate_q):
    w = synth.make_fmt_weights(cfg, 0)
    x60, cond = _inputs(cfg)
    s = _sampler(cfg, w)
    v = s.forward(x60, cond, 0.4444444)
    assert np.array_equal(v, s.forward(x60, cond, 0.4444444))
    c = cosine(v, torch_lia.TorchFmt(cfg, w).forward(x60, cond, 0.4444444))
    cq = cosine(v, QuantFmt(cfg, w).forward(x60, cond, 0.4444444))
    print(f"8-bit forward: cosine {c:.5f} to float64, {cq:.6f} to the quantised operands")
    assert c > gate
    assert cq > gate_q
    s.close()


@pytest.mark.parametrize("sinks", [0, 10])
def test_chunk_is_its_forwards(sinks):
    """a captured chunk of one Euler step against a single forward of the
    same handle: the same kernels on the same rows, so only the step's own
    float32 arithmetic differs (a few 2^-24 of the terms it adds)"""
    cfg = dict(synth.FMT_SMALL, nfe=2)
    w = synth.make_fmt_weights(cfg, 0)
    io = synth.make_fmt_chunk(cfg, 0)
    s = _sampler(cfg, w)
    s.set_sinks(sinks)
    got = s.sample(io["wr"], io["prev_wa"], io["cond_audio"], io["prev_x"], io["x0"], io["emotion"])
    assert np.array_equal(got, s.sample(io["wr"], io["prev_wa"], io["cond_audio"], io["prev_x"], io["x0"], io["emotion"]))
    D, P, CF, nfe = cfg["dim_w"], cfg["prev_frames"], cfg["chunk_frames"], cfg["nfe"]
    cond = np.zeros((3, P + CF, D + cfg["dim_a"] + cfg["dim_e"]), np.float32)
    for b in range(3):
        for f in range(P + CF):
            cond[b, f, :D] = io["wr"]
            if not (b == 0 and f >= P):
                cond[b, f, D:2 * D] = io["prev_wa"][f] if f < P else io["cond_audio"][f - P]
            if b == 1:
                cond[b, f, D + cfg["dim_a"] + io["emotion"]] = 1.0
    x = io["x0"].astype(np.float32)
    for i in range(nfe - 1):
        t0, t1 = np.float32(i / (nfe - 1)), np.float32((i + 1) / (nfe - 1))
        v = s.forward(np.concatenate([io["prev_x"], x]), cond, float(t0))
        x = x + (t1 - t0) * ((v[0] + np.float32(cfg["a_cfg"]) * (v[2] - v[0])) + np.float32(cfg["e_cfg"]) * (v[1] - v[2]))[P:]
    np.testing.assert_allclose(got, x, rtol=2e-6, atol=2e-6 * float(np.abs(v).max()))
    s.close()


def test_memory_and_refusals():
    """the 8-bit weights take less device memory than the f16 ones; widths
    that the 8-bit product cannot address are refused"""
    cfg = synth.FMT_CONFIG
    w = synth.make_fmt_weights(cfg, 0)
    used = {}
    for dt in (tpmd.DTYPE_F16, tpmd.DTYPE_F8):
        torch.cuda.synchronize()
        a = torch.cuda.mem_get_info()[0]
        s = _sampler(cfg, w, dt)
        used[dt] = a - torch.cuda.mem_get_info()[0]
        s.close()
    # depth (3 + 8) dim_h^2 + (6 depth + 2) dim_h^2 weights at a byte less each
    # (allocations come in 2 MB pages; the quantised rows take about 2 MB)
    assert used[tpmd.DTYPE_F16] - used[tpmd.DTYPE_F8] > (cfg["depth"] * 17 + 2) * cfg["dim_h"] ** 2 - 12e6
    with pytest.raises(tpmd.TpmdError, match="multiples of 16"):
        tpmd.FmtSampler(dict(synth.FMT_SMALL, dim_h=264, n_heads=4), 0, tpmd.DTYPE_F8)
