"""The router where its numbers and its loop can go wrong: entries that another lane fills in, several rows per warp, scores far from
the largest one, logits far below zero.  Against the 64-bit form of tests/plain_forms.py."""
import itertools

import pytest
import torch

from tests import plain_forms as P
from tests.test_gpu_router import check_backward, check_forward, logits_of

pytestmark = pytest.mark.gpu

U = P.U32


@pytest.mark.parametrize("E,K", [(60, 6), (129, 7), (256, 8), (700, 32)])
@pytest.mark.parametrize("score,renorm", list(itertools.product(["softmax", "sigmoid"], [True, False])))
def test_a_warps_first_row_has_the_score_sums_gradient(score, renorm, E, K):
    """The picks' gradients are added to d_score_sums entries that other lanes have filled in: one row per warp, so that every row
    is a warp's first, and runs agree."""
    from mok import functional as F
    cfg = F.MoKRouterConfig(topk=K, score=score, renormalize=renorm)
    logits = logits_of(1500, E, torch.float32, seed=E)
    r = check_forward(cfg, logits)
    first = check_backward(cfg, logits, r)
    for _ in range(10):
        assert torch.equal(check_backward(cfg, logits, r), first)


def spread_logits(T, E, far, seed, step=0.25):
    """fp32 logits on multiples of `step`, so that differences of two are exact, from 0 down to -far."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    l = -torch.randint(0, int(far / step) + 1, (T, E), generator=gen, device="cuda").float() * step
    l[:, 0] = 0.0
    return l


@pytest.mark.parametrize("renorm", [True, False], ids=["share", "score"])
def test_softmax_far_below_the_largest_logit(renorm):
    """The error of a score does not grow with its distance from the row's largest: an exp (4 half-steps), a sum of at most E of them
    (4 and 7 additions for 8 experts: a lane's four slots, a tree of five over the warp, 9 at most), a quotient, `scale` (1): 16."""
    from mok import functional as F
    E = K = 8
    logits = spread_logits(4000, E, 80.0, seed=1)
    r = F.route(F.MoKRouterConfig(topk=K, renormalize=renorm), logits, balance=True)
    picked, weights, _, sums, s, _ = P.route(logits, K, "softmax", None, renorm)
    assert torch.equal(r.top_experts, picked)
    off = (r.router_weights.double() - weights).abs() / (U * weights)
    assert off.max() <= 16, off.max()
    # a warp adds at most ceil(T / warps) rows, a block its warps, the reduction its blocks: below 200 additions of positive numbers
    assert ((r.score_sums.double() - sums).abs() <= (16 + 200) * U * sums).all()


@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
def test_sigmoid_over_its_range(bias):
    """Scores of logits from -100 to 100, fp32's subnormal numbers included: an exp, a sum, a quotient, a product: 8 half-steps, and
    half a step of the smallest number."""
    from mok import functional as F
    E = K = 16
    logits = spread_logits(2000, E, 200.0, seed=2) + 100.0
    b = torch.zeros(E, device="cuda") if bias else None
    r = F.route(F.MoKRouterConfig(topk=K, score="sigmoid", renormalize=False), logits, b)
    want = torch.sigmoid(logits.double()).gather(1, r.top_experts)
    assert ((r.router_weights.double() - want).abs() <= 8 * U * want + 2.0 ** -149).all()


@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("level", [-80.0, -90.0, -100.0, -110.0, -300.0, -600.0])
def test_shares_of_sigmoid_scores_far_below_zero(level, dtype, bias):
    """Renormalised weights are shares of the scores' sum however small the scores are: the token keeps its experts, and the gradient
    its slope.  A share: two exps, a quotient each, a product (12), a sum of K (5), a quotient (1), `scale` (1)."""
    from mok import functional as F
    E, K = 32, 6
    logits = (level + spread_logits(300, E, 12.0, seed=3, step=0.5)).to(dtype)      # (halves, exact in bf16 only near zero: as rounded)
    b = torch.zeros(E, device="cuda")
    b[::4] = 0.25
    b = b if bias else None
    cfg = F.MoKRouterConfig(topk=K, score="sigmoid", scale=2.5)
    r = F.route(cfg, logits, b)
    picked, weights, _, _, _, _ = P.route(logits, K, "sigmoid", b, True, 2.5)
    assert torch.equal(r.top_experts, picked)
    assert ((r.router_weights.double() - weights).abs() <= 20 * U * weights + 2.0 ** -149).all()
    assert ((r.router_weights.double().sum(1) - 2.5).abs() <= 2.5 * (20 + K) * U).all()
    dw = torch.randn(300, K, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    d = F.route_backward(cfg, logits, r, dw)
    want = P.route_bwd(logits, picked, dw, None, "sigmoid", True, 2.5)
    # share * (dw - mean): dw and the mean, each off by 30 roundings of itself, the share by 20
    share = weights / 2.5
    terms = 2.5 * share * (dw.double().abs() + (share * dw.double().abs()).sum(1, keepdim=True))
    room = torch.zeros_like(want).scatter_(1, picked, 64 * U * terms) + 2.0 ** -149
    if dtype == torch.bfloat16:
        room = room + P.U16 * (want.abs() + room)
    assert ((d.double() - want).abs() <= room).all()
