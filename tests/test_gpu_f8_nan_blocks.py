"""Blocks of nothing but NaN: a NaN does not count in its block's maximum, so
such a block has the smallest scale, 2^-126, in the quantiser's two forms and
in the 8-bit output of the product's two tile sizes."""
import pytest
import torch

import tpmd
from test_gpu_f8 import padded, quant_ref, quantised, same_bytes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("M,K,extra", [(1, 128, 0), (3, 256, 0), (200, 300, 0), (130, 129, 1), (2, 1, 0), (1500, 4096, 0)])
def test_quantiser(M, K, extra, dtype, rows):
    """one block, whole rows, a last block of one column; rows off vector
    boundaries; enough rows for four loads in flight"""
    g = torch.Generator().manual_seed(M + K)
    x = torch.randn(M, K + extra, generator=g)[:, extra:]
    x[:, :128] = float("nan")
    x[M // 2:] = float("nan")
    x = x.to(dtype)
    q, _ = padded(M, K)
    s = torch.zeros(-(-M // rows), -(-K // 128), device="cuda")
    d = torch.empty(M, K + extra, dtype=dtype, device="cuda")[:, extra:]
    d.copy_(x)
    tpmd.quant_f8(d, q, s, rows=rows)
    rq, rs = quant_ref(x, rows)
    assert bool((rs == 2.0 ** -126).any())
    assert torch.equal(s.cpu(), rs) and same_bytes(q, rq)


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("M,N,K", [(60, 256, 256), (180, 300, 1024), (2400, 2304, 128), (2400, 2306, 72)])
def test_product(M, N, K, act):
    """a NaN in a row of X makes every column of that row NaN"""
    g = torch.Generator().manual_seed(K)
    X, sx = quantised(M, K, 1, g)
    W, sw = quantised(N, K, 128, g, scale=K ** -0.5)
    X.view(torch.uint8)[[0, M // 2, M - 1], K // 3] = 0x7F
    bias = torch.randn(N, generator=g).cuda()
    Y = torch.empty(M, N, device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, Y, bias=bias, act=act)
    q, _ = padded(M, N)
    sy = torch.zeros(M, -(-N // 128), device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, q, sy=sy, bias=bias, act=act)
    tpmd.tpk_status()
    assert bool(Y[M // 2].isnan().all()) and not bool(Y[1].isnan().any())
    rq, rs = quant_ref(Y.cpu(), 1)
    assert torch.equal(sy.cpu(), rs) and same_bytes(q, rq)
