"""f16 attention over very many keys that each weigh next to nothing beside
the largest: together they count.

The weights go through f16 into the product with v, 2^7 of them to the
largest weight that the running maximum knows: off by 2^-11 relative down to
2^-21 of that largest one, by 2^-32 of it below (half of f16's smallest step,
2^-25, over 2^7). With p the float64 weights (sum 1), top the largest, A =
sum_j p_j |v_j|, an output is off by at most 2^-11 A + keys 2^-32 top max |v|,
its own rounding (2^-11 |o|, 2^-25) and the f32 terms: scores off by
d = (D + 4) 2^-23 x, x the row's largest scale sum |q k|, so weights by 2 d
relative, 2^-20 for exponentials, 2^-23 a key for the sums."""
import pytest
import torch

import tpmd

pytestmark = pytest.mark.gpu


def check(q, k, v, scale, left=-1, right=-1, sinks=0):
    (B, Tq, Hq, D), (Tk, Hkv) = q.shape, k.shape[1:3]
    out = torch.empty_like(q)
    tpmd.attn_window(q, k, v, out, left, right, sinks, scale=scale)
    tpmd.tpk_status()
    g = Hq // Hkv
    for b in range(B):
        for h in range(Hq):
            qq, kk, vv = (t.double() for t in (q[b, :, h], k[b, :, h // g], v[b, :, h // g]))
            pos = torch.arange(Tq, device="cuda")[:, None] + Tk - Tq
            j = torch.arange(Tk, device="cuda")[None, :]
            ok = (j >= 0) & (pos >= 0)
            if right >= 0:
                ok = ok & (j <= pos + right)
            if left >= 0:
                ok = ok & ((j >= pos - left) | (j < sinks))
            p = torch.softmax((qq @ kk.t() * scale).masked_fill(~ok, -float("inf")), dim=1)
            o, A = p @ vv, p @ vv.abs()
            x = (qq.abs() @ kk.abs().t() * scale).amax(dim=1, keepdim=True)
            e = A * (2 * (D + 4) * 2.0 ** -23 * x + 2.0 ** -20 + Tk * 2.0 ** -23 + 2.0 ** -11)
            e = e + Tk * 2.0 ** -32 * p.amax(dim=1, keepdim=True) * vv.abs().max() + 2.0 ** -11 * o.abs() + 2.0 ** -25
            err = (out[b, :, h].double() - o).abs()
            assert bool((err <= e).all()), (h, float((err / e).max()))


# powers of two that the other keys weigh less than the large one
LESS = [18.4, 22.0, 24.5, 25.0, 27.0, 30.0]


@pytest.mark.parametrize("at", [0, 30000, 60000])
@pytest.mark.parametrize("less", LESS)
def test_one_token_over_many_keys(less, at):
    """keys shared out over warpgroups and CTAs; the large key among the
    first, in the middle, the last. Its v is 0, so the rest is the output"""
    T, D = 60001, 64
    g = torch.Generator().manual_seed(int(less * 10))
    q = torch.zeros(1, 1, 2, D)
    q[..., 0] = 1.0
    k = torch.zeros(1, T, 1, D)
    k[:, at, :, 0] = less
    v = 1.0 + 0.25 * torch.randn(1, T, 1, D, generator=g)
    v[:, at] = 0.0
    check(*(t.half().cuda() for t in (q, k, v)), scale=0.6931471805599453)


@pytest.mark.parametrize("less", LESS)
@pytest.mark.parametrize("D", [64, 128])
def test_prompts(less, D):
    """two row tiles a CTA; windows with a large key among the sinks, and
    rows whose window has one of its own"""
    T, H = 2500, 80
    g = torch.Generator().manual_seed(D)
    q = torch.zeros(1, T, H, D)
    q[..., 0] = 1.0
    k = torch.zeros(1, T, H, D)
    k[:, 1, :, 0] = less
    k[:, 1777, : H // 2, 0] = less
    v = 1.0 + 0.25 * torch.randn(1, T, H, D, generator=g)
    v[:, [1, 1777]] = 0.0
    check(*(t.half().cuda() for t in (q, k, v)), scale=0.6931471805599453, left=2000, right=0, sinks=4)


def test_rising_scores_stay_within_f16():
    """every tile raises the maximum by a little less than the threshold at
    which the weights' reference moves, and by a little more"""
    T, D = 4096, 64
    q = torch.zeros(1, 1, 2, D)
    q[..., 0] = 1.0
    for step in (0.12, 7.9 / 64, 8.1 / 64, 0.25, 1.0):
        k = torch.zeros(1, T, 1, D)
        k[0, :, 0, 0] = torch.arange(T).float() * step
        v = torch.randn(1, T, 1, D, generator=torch.Generator().manual_seed(3))
        check(*(t.half().cuda() for t in (q, k, v)), scale=0.6931471805599453)
