"""The sampler's attention beyond the band kernel: wide windows, first frames
that stay visible, wide heads (tpfm_*, tpfm_set_sinks), against the float64
torch DiT with the same mask, and whole chunks captured as one graph."""
import numpy as np
import pytest
import torch

import oracle as O
import torch_lia
import tpmd
from metrics import cosine
from tpmd import synth

pytestmark = pytest.mark.gpu


def _inputs(cfg, seed=1):
    rng = np.random.default_rng(seed)
    T = cfg["chunk_frames"] + cfg["prev_frames"]
    CD = cfg["dim_w"] + cfg["dim_a"] + cfg["dim_e"]
    return (rng.standard_normal((T, cfg["dim_w"])).astype(np.float32),
            rng.standard_normal((3, T, CD)).astype(np.float32))


def _sampler(cfg, w, dtype, sinks=0):
    s = tpmd.FmtSampler(cfg, 0, dtype)
    s.set_tensors(w)
    s.set_sinks(sinks)
    s.prepare()
    return s


def _torch_forward(cfg, w, sinks, x60, cond, t):
    """|i - j| <= window, or j < sinks and not past the window's right end"""
    T = cfg["chunk_frames"] + cfg["prev_frames"]
    i, j = torch.arange(T)[:, None], torch.arange(T)[None, :]
    reach = torch.where((j < sinks) & (j <= i + cfg["attn_window"]), T, cfg["attn_window"])
    return torch_lia.TorchFmt(dict(cfg, attn_window=reach), w).forward(x60, cond, t)


CASES = [(dict(synth.FMT_SMALL, attn_window=8), 0), (dict(synth.FMT_SMALL, attn_window=59), 0),
         (dict(synth.FMT_SMALL, attn_window=100000), 0), (dict(synth.FMT_SMALL, attn_window=2), 10),
         (dict(synth.FMT_SMALL, attn_window=0), 1), (dict(synth.FMT_SMALL, attn_window=12, n_heads=2), 3),
         (dict(synth.FMT_SMALL, attn_window=2, n_heads=1), 0), (dict(synth.FMT_SMALL, attn_window=9, n_heads=1), 60)]


@pytest.mark.parametrize("cfg,sinks", CASES, ids=lambda c: str(c) if isinstance(c, int) else f"w{c['attn_window']}h{c['n_heads']}")
def test_forward_matches_float64(cfg, sinks):
    """f32: the gates of the banded forward; f16: cosine as in its chunk test"""
    w = synth.make_fmt_weights(cfg, 0)
    x60, cond = _inputs(cfg)
    r = _torch_forward(cfg, w, sinks, x60, cond, 0.4444444)
    s = _sampler(cfg, w, tpmd.DTYPE_F32, sinks)
    v = s.forward(x60, cond, 0.4444444)
    assert cosine(v, r) > 1 - 1e-6
    assert np.abs(v - r).max() < 1e-3 * np.abs(r).max()
    s.close()
    s = _sampler(cfg, w, tpmd.DTYPE_F16, sinks)
    assert cosine(s.forward(x60, cond, 0.4444444), r) > 0.999
    s.close()


@pytest.mark.parametrize("dtype", [tpmd.DTYPE_F32, tpmd.DTYPE_F16])
def test_chunk_with_a_wide_window(dtype):
    """the first call captures the graph; replays give the same bits; the
    oracle has the same window"""
    cfg = dict(synth.FMT_SMALL, attn_window=20)
    w = synth.make_fmt_weights(cfg, 0)
    io = synth.make_fmt_chunk(cfg, 0)
    args = (io["wr"], io["prev_wa"], io["cond_audio"], io["prev_x"], io["x0"], io["emotion"])
    s = _sampler(cfg, w, dtype)
    got = s.sample(*args)
    assert np.array_equal(got, s.sample(*args))
    ref = O.Fmt(cfg, w).sample(*args)
    assert cosine(got, ref) > (1 - 1e-6 if dtype == tpmd.DTYPE_F32 else 0.999)
    # sinks change the chunk, and taking them back gives the first bits again
    s.set_sinks(10)
    other = s.sample(*args)
    assert not np.array_equal(got, other)
    s.set_sinks(0)
    assert np.array_equal(got, s.sample(*args))
    s.close()


def test_band_is_untouched():
    """sinks that add nothing (the band already reaches them all) agree with
    the band kernel to float32 accuracy, and the band itself does not use
    them"""
    cfg = dict(synth.FMT_SMALL, chunk_frames=4, prev_frames=2, attn_window=7)
    w = synth.make_fmt_weights(cfg, 0)
    x60, cond = _inputs(cfg)
    s = _sampler(cfg, w, tpmd.DTYPE_F32)
    a = s.forward(x60, cond, 0.5)
    s.set_sinks(6)
    b = s.forward(x60, cond, 0.5)
    assert cosine(a, b) > 1 - 1e-9
    s.close()


def test_refusals():
    s = tpmd.FmtSampler(synth.FMT_SMALL, 0)
    for bad in (-1, 61):
        with pytest.raises(tpmd.TpmdError, match="sinks"):
            s.set_sinks(bad)
    s.set_sinks(60)
    s.close()
    with pytest.raises(tpmd.TpmdError, match="invalid config"):
        tpmd.FmtSampler(dict(synth.FMT_SMALL, attn_window=-1), 0)
