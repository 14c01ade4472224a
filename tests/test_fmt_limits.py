"""Attention windows and head widths at the ends of their ranges
(tpfm_create): an unlimited window, as INT_MAX means it, sees every frame; a
head wider than the attention kernels take is refused at creation."""
import numpy as np
import pytest

import torch_lia
import tpmd
from metrics import cosine
from tpmd import synth


def _forward(cfg, w, dtype):
    rng = np.random.default_rng(1)
    T = cfg["chunk_frames"] + cfg["prev_frames"]
    x60 = rng.standard_normal((T, cfg["dim_w"])).astype(np.float32)
    cond = rng.standard_normal((3, T, cfg["dim_w"] + cfg["dim_a"] + cfg["dim_e"])).astype(np.float32)
    s = tpmd.FmtSampler(cfg, 0, dtype)
    s.set_tensors(w)
    s.prepare()
    v = s.forward(x60, cond, 0.4444444)
    s.close()
    return v, torch_lia.TorchFmt(dict(cfg, attn_window=min(cfg["attn_window"], T)), w).forward(x60, cond, 0.4444444)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [60, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 7, 2 ** 31 - 1])
@pytest.mark.parametrize("dtype", [tpmd.DTYPE_F32, tpmd.DTYPE_F16])
def test_unlimited_windows(window, dtype):
    """2 window + 1 leaves the ints from 2^30 on"""
    cfg = dict(synth.FMT_SMALL, attn_window=window)
    v, r = _forward(cfg, synth.make_fmt_weights(cfg, 0), dtype)
    # the gates of the banded forward
    assert cosine(v, r) > (1 - 1e-6 if dtype == tpmd.DTYPE_F32 else 0.999)


@pytest.mark.gpu
def test_the_widest_head_runs():
    cfg = dict(synth.FMT_SMALL, dim_h=256, n_heads=1)
    v, r = _forward(cfg, synth.make_fmt_weights(cfg, 0), tpmd.DTYPE_F32)
    assert cosine(v, r) > 1 - 1e-6


@pytest.mark.parametrize("dim_h,n_heads", [(264, 1), (1024, 2), (528, 2)])
@pytest.mark.parametrize("dtype", [tpmd.DTYPE_F32, tpmd.DTYPE_F16, tpmd.DTYPE_F8])
def test_wider_heads_are_refused(dim_h, n_heads, dtype):
    """on the host, before a device is looked for"""
    with pytest.raises(tpmd.TpmdError, match="head"):
        tpmd.FmtSampler(dict(synth.FMT_SMALL, dim_h=dim_h, n_heads=n_heads), 0, dtype)
