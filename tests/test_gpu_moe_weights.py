"""How exact routing's weights are, for logits near each other and far apart.

With u = 2^-24, half a step of fp32.  A softmax score: exp is off by a step (2 u), what the difference lacks is made up for (u for the addition), the sum by its
rounding (u) and its terms', the quotient by u.  The terms come of the hardware's exp, off by 2 u and by 1.5 u d for one that is d below the largest; weighted with
the scores that is at most 2 u + 1.5 u ln 1024.  So 19 u.  A sigmoid: 2 u of exp, an addition, a quotient: 4 u.  Divided by their sum the sum over all experts cancels: 4 u of a
score, as much of the sum's terms, four additions of up to 16, 1e-20 and a quotient: 14 u.  The factor behind it: u.

Where fp32 ends: a softmax score below 2^-126 is a multiple of 2^-149, off by less than 2^-148; exp(-l) of a sigmoid is infinite from l = -88.8 on, the score, which is then
below 2^-127, zero.  What is divided by the scores' sum later is off by that much more."""
import pytest
import torch

from nnfusion_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _weights(logits, experts, score, renormalize, scale):
    x = logits.double()
    s = torch.softmax(x, 1) if score == "softmax" else 1 / (1 + torch.exp(-x))
    w = s.gather(1, experts.long())
    by = w.sum(1, keepdim=True) + 1e-20 if renormalize else torch.ones_like(w[:, :1])
    return w / by * scale, 2.0 ** (-148 if score == "softmax" else -127) / by * scale + 2.0 ** -149


@pytest.mark.parametrize("tokens,n,k", [(1, 256, 8), (16, 64, 16), (500, 128, 8), (3000, 60, 4), (700, 512, 10), (9, 1024, 16), (300, 1024, 16)])
@pytest.mark.parametrize("score,with_bias", [("softmax", False), ("softmax", True), ("sigmoid", False), ("sigmoid", True)])
@pytest.mark.parametrize("spread", [0.01, 1.5, 20.0, 60.0])
def test_weights(gpu, tokens, n, k, score, with_bias, spread):
    gen = torch.Generator().manual_seed(tokens + n)
    # (whole and odd numbers of steps, so that differences are not exact)
    logits = (spread * torch.randn((tokens, n), generator=gen) + 3.3).to(gpu)
    bias = (torch.rand((n,), generator=gen) * 2).to(gpu) if with_bias else None
    for renormalize in (True, False):
        for scale in (1.0, 2.5):
            got, experts, *_ = ops.moe_route(logits, k, score=score, bias=bias, renormalize=renormalize, scale=scale)
            want, least = _weights(logits, experts, score, renormalize, float(scale))
            bound = (15 if renormalize else 20 if score == "softmax" else 5) * U
            off = (got.double() - want).abs()
            assert bool((off <= bound * want.abs() + least).all()), (((off - least) / want).max() / U, renormalize, scale)


def test_logits_at_both_ends_of_fp32(gpu):
    most = torch.finfo(torch.float32).max
    logits = torch.tensor([[most, -most, 0.0, most], [-most, -most, -most, -most], [float("inf"), most, 1.0, float("-inf")], [1e30, 1e30, -1e30, 3.0]], device=gpu)
    for tokens in (4, 400):
        x = logits.repeat(tokens // 4, 1)
        weights, experts, *_ = ops.moe_route(x, 4, renormalize=False)
        want = torch.tensor([[0.5, 0.5, 0, 0], [0.25] * 4, [0.5, 0.5, 0, 0], [0.5, 0.5, 0, 0]], device=gpu).repeat(tokens // 4, 1)
        assert torch.equal(weights, want)
