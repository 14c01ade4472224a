"""The 8-bit output of tpk_gemm_f8 where N ends inside a block of 128: the
last block's scale is that of the columns that exist. The 8-bit output equals
the quantised f32 output, bit for bit (the same sums, the same quantisation),
whatever bias stands in the last column, on 128 x 128 and 256 x 256 tiles."""
import pytest
import torch

import tpmd
from test_gpu_f8 import padded, quant_ref, quantised, same_bytes

pytestmark = pytest.mark.gpu


def both_outputs(M, N, K, act, bias, seed=0):
    g = torch.Generator().manual_seed(seed + M + 3 * N + 7 * K)
    X, sx = quantised(M, K, 1, g)
    W, sw = quantised(N, K, 128, g, scale=K ** -0.5)
    b = bias(torch.randn(N, generator=g)).cuda()
    Y = torch.full((M, N), float("nan"), device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, Y, bias=b, act=act)
    q, raw = padded(M, N, extra=16)
    sy = torch.full((M, -(-N // 128)), -1.0, device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, q, sy=sy, bias=b, act=act)
    tpmd.tpk_status()
    assert bool((raw[:, N:] == 0x7F).all())
    return Y.cpu(), q, sy.cpu()


def last(value):
    def bias(b):
        b[-1] = value
        return b
    return bias


# the last three fill no SMs with tiles of 256 x 256
SHAPES = [(2400, 2306, 72), (19000, 129, 128), (2310, 2305, 136), (2560, 2049, 264), (5000, 1100, 144), (2400, 2304, 72),
          (180, 129, 300), (777, 1000, 528), (60, 257, 1040)]


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_last_block(M, N, K, act):
    for bias in (lambda b: b, last(40.0), last(-40.0)):
        Y, q, sy = both_outputs(M, N, K, act, bias)
        rq, rs = quant_ref(Y, 1)
        assert torch.equal(sy, rs) and same_bytes(q, rq)


@pytest.mark.parametrize("act", [0, 2])
def test_a_last_column_that_its_bias_cancels(act):
    """sums that the last column's bias takes back: the block is all but zero"""
    M, N, K = 2400, 2305, 128
    g = torch.Generator().manual_seed(9)
    X, sx = quantised(M, K, 1, g)
    W, sw = quantised(N, K, 128, g)
    # the last row of W and all of X: 8 x 8 x 128 scales apart, minus its bias
    X.copy_(torch.full((M, K), 8.0).to(X.dtype))
    sx.fill_(2.0 ** -6)
    W[-1].copy_(torch.full((K,), 8.0).to(W.dtype))
    sw[-1] = 2.0 ** -6
    b = torch.zeros(N, device="cuda")
    b[-1] = -(2.0 + 2.0 ** -10)  # 8 x 8 x 128 x 2^-12 = 2
    q, _ = padded(M, N)
    sy = torch.empty(M, 19, device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, q, sy=sy, bias=b, act=act)
    Y = torch.empty(M, N, device="cuda")
    tpmd.gemm_f8(X, sx, W, sw, Y, bias=b, act=act)
    tpmd.tpk_status()
    if act == 0:
        assert bool((Y[:, -1] == -2.0 ** -10).all()) and bool((sy[:, -1] == 2.0 ** -10 / 448).all())
        assert bool((q[:, -1].float() == -448.0).all())
    rq, rs = quant_ref(Y.cpu(), 1)
    assert torch.equal(sy.cpu(), rs) and same_bytes(q, rq)
