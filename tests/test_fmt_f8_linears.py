"""The sampler's 8-bit linears one at a time (TPMD_DTYPE_F8), so that a wrong
scale of a single block of 128 x 128 weights shows.

A DiT of one block whose weights leave one path open: everything beside the
linear under test is zero, one or the identity, the residual is small, and the
decoder is the identity. A quantised operand is off by at most 2^-4 / sqrt(3) =
0.036 of its value rms, a product of two by 0.051; linears in a row add in
squares, tanh GELU passes an error on by a factor below 1.13, a softmax passes
the scores' error d on as d rms(v) / rms(o). The gate stands over each group of
128 output columns, the columns of one block of weights. The CPU test shows
that the DiT with operands quantised in float64 keeps to the gates and that it
does not once a single block's scale is doubled."""
import numpy as np
import pytest
import torch

import torch_lia
import tpmd
from test_gpu_fmt_f8 import QuantFmt
from tpmd import synth

E = 0.051
WIDTHS = [256, 1024]
# path: the weights it opens, linears on it in squares, key window
PATHS = {
    "v": ("qkv", E, 0),
    "qk": ("qkv", E * (1 + 2 * 1.7 ** 2) ** 0.5, 2),  # scores of variance 1, rms(v) / rms(o) < 1.7 over five keys
    "mlp": ("mlp", E * (1.13 ** 2 + 1) ** 0.5, 0),
    "gate1": ("mod", E, 0), "gate2": ("mod", E, 0), "shift": ("mod", E, 0), "scale": ("mod", E, 0),
    "mod1": ("mod+qkv", E * 2 ** 0.5, 0),
    "mod2": ("mod+mlp", E * (2 * 1.13 ** 2 + 1) ** 0.5, 0),
}


def config(H, path):
    return dict(synth.FMT_SMALL, dim_h=H, n_heads=H // 64, depth=1, dim_w=H, dim_a=64, attn_window=PATHS[path][2])


def weights(cfg, path):
    H = cfg["dim_h"]
    rng = np.random.default_rng([H, sorted(PATHS).index(path)])
    w = {n: np.zeros(s, np.float32) for n, s in synth.fmt_shapes(cfg).items()}

    def rand(*s):
        return (rng.standard_normal(s) / s[1] ** 0.5).astype(np.float32)

    w["decoder.linear.weight"] = np.eye(H, dtype=np.float32)
    w["pos_embed"] = (0.05 * rng.standard_normal(w["pos_embed"].shape)).astype(np.float32)
    ada, last, b = "blocks.0.adaLN_modulation.1", "decoder.adaLN_modulation.1", "blocks.0."
    # (silu halves what it gets: conditions of about one)
    w["c_embedder.weight"] = 2.0 * rand(*w["c_embedder.weight"].shape)
    rows = {"shift1": 0, "scale1": 1, "gate1": 2, "shift2": 3, "scale2": 4, "gate2": 5}

    def modulate(name, table=ada):
        at = rows[name] * H
        w[table + ".weight"][at:at + H] = 1.5 * rand(H, H)

    gates = w[ada + ".bias"].reshape(6, H)
    if path in ("v", "qk", "mod1"):
        gates[2] = 1.0
        w[b + "attn.qkv.weight"] = rand(3 * H, H)
        w[b + "attn.proj.weight"] = np.eye(H, dtype=np.float32)
    if path in ("mlp", "mod2"):
        gates[5] = 1.0
        w[b + "mlp.fc1.weight"], w[b + "mlp.fc2.weight"] = rand(4 * H, H), 2.0 * rand(H, 4 * H)
    if path in ("mod1", "mod2"):
        modulate("shift" + path[3])
        modulate("scale" + path[3])
    if path == "gate1":
        modulate("gate1")
        w[b + "attn.proj.bias"][:] = 1.0
    if path == "gate2":
        modulate("gate2")
        w[b + "mlp.fc2.bias"][:] = 1.0
    if path in ("shift", "scale"):
        rows.update(shift=0, scale=1)
        modulate(path, last)
    return w


def inputs(cfg):
    rng = np.random.default_rng(7)
    T = cfg["chunk_frames"] + cfg["prev_frames"]
    return (rng.standard_normal((T, cfg["dim_w"])).astype(np.float32),
            rng.standard_normal((3, T, cfg["dim_w"] + cfg["dim_a"] + cfg["dim_e"])).astype(np.float32), 0.4444444)


def worst(got, want):
    """largest error of a group of 128 columns, of that group's norm"""
    d, w = (np.asarray(x, np.float64).reshape(-1, want.shape[-1] // 128, 128) for x in (got - want, want))
    return float((np.sqrt((d ** 2).sum((0, 2))) / np.sqrt((w ** 2).sum((0, 2)))).max())


def open_weights(cfg, w, path):
    """the 8-bit matrices on the path: name, and the rows of it that are not zero, in blocks"""
    names = {"qkv": ["blocks.0.attn.qkv.weight"], "mlp": ["blocks.0.mlp.fc1.weight", "blocks.0.mlp.fc2.weight"],
             "mod": ["blocks.0.adaLN_modulation.1.weight", "decoder.adaLN_modulation.1.weight"]}
    for part in PATHS[path][0].split("+"):
        for n in names[part]:
            live = np.abs(w[n]).reshape(-1, 128, w[n].shape[1]).max((1, 2)) > 0
            if "qkv" in n and PATHS[path][2] == 0:
                live[:2 * cfg["dim_h"] // 128] = False  # (one key: its weight is one whatever q and k are)
            if path == "qk":
                live[2 * cfg["dim_h"] // 128:] = False
            if live.any():
                yield n, np.flatnonzero(live)


@pytest.mark.parametrize("path", list(PATHS))
def test_gates_hold_and_find_a_wrong_block(path):
    """in float64 on the CPU: the quantised DiT within the gate; with one
    block's scale doubled, at either end of each matrix, beyond it"""
    cfg = config(256, path)
    w = weights(cfg, path)
    at = inputs(cfg)
    want = torch_lia.TorchFmt(cfg, w).forward(*at)
    gate = PATHS[path][1]
    e = worst(QuantFmt(cfg, w).forward(*at), want)
    print(f"{path}: {e:.4f} of {gate:.4f}")
    assert 0.2 * gate < e < gate
    for n, blocks in open_weights(cfg, w, path):
        for r, k in ((blocks[0], 0), (blocks[-1], w[n].shape[1] // 128 - 1)):
            bad = QuantFmt(cfg, w)
            bad.w[n] = bad.w[n].clone()
            bad.w[n][128 * r:128 * r + 128, 128 * k:128 * k + 128] *= 2.0
            e = worst(bad.forward(*at), want)
            print(f"  {n} block {r}, {k} doubled: {e:.4f}")
            assert e > gate


@pytest.mark.gpu
@pytest.mark.parametrize("H", WIDTHS)
@pytest.mark.parametrize("path", list(PATHS))
def test_linear(path, H):
    cfg = config(H, path)
    w = weights(cfg, path)
    at = inputs(cfg)
    want = torch_lia.TorchFmt(cfg, w).forward(*at)
    s = tpmd.FmtSampler(cfg, 0, tpmd.DTYPE_F8)
    s.set_tensors(w)
    s.prepare()
    e = worst(s.forward(*at), want)
    s.close()
    print(f"{path}, {H} wide: {e:.4f} of {PATHS[path][1]:.4f}")
    assert e < PATHS[path][1]
