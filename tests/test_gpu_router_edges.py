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


@pytest.mark.parametrize("level", [-640.0, -700.0, -720.0, -735.0, -742.0, -744.5, -746.0, -800.0, -1e30])
def test_shares_at_the_end_of_the_sigmoids_range(level):
    """Rows whose largest pick's score is just inside 64 bits' range (exp(-745)) have shares and a gradient, rows beyond have none; never
    a NaN or an infinity.  One share per distance from the largest: the expected ones are exp of it, over their sum."""
    from mok import functional as F
    E = K = 4
    below = torch.tensor([0.0, 0.25, 0.5, 0.0], device="cuda")
    logits = (level - below).expand(8, E).contiguous()
    cfg = F.MoKRouterConfig(topk=K, score="sigmoid")
    r = F.route(cfg, logits, balance=True)
    dw = torch.randn(8, K, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    d = F.route_backward(cfg, logits, r, dw, torch.ones(E, device="cuda"))
    assert torch.isfinite(r.router_weights).all() and torch.isfinite(d).all()
    if level < -745:
        assert (r.router_weights == 0).all() and (d == 0).all()
        return
    share = torch.softmax(logits.double(), 1).gather(1, r.top_experts)
    assert ((r.router_weights.double() - share).abs() <= 20 * U * share).all()
    want = share * (dw.double() - (share * dw.double()).sum(1, keepdim=True))
    size = share * (dw.double().abs() + (share * dw.double().abs()).sum(1, keepdim=True))
    assert ((d.double().gather(1, r.top_experts) - want).abs() <= 64 * U * size).all()


@pytest.mark.parametrize("renorm", [True, False], ids=["share", "score"])
def test_sigmoid_gradient_near_one(renorm):
    """Logits up to 40: 1 - s is a small number of its own, not what is left of 1 after s is rounded."""
    from mok import functional as F
    E, K = 24, 4
    logits = spread_logits(500, E, 35.0, seed=5) + 40.0
    cfg = F.MoKRouterConfig(topk=K, score="sigmoid", renormalize=renorm)
    r = F.route(cfg, logits)
    gen = torch.Generator(device="cuda").manual_seed(6)
    dw, ds = torch.randn(500, K, generator=gen, device="cuda"), torch.randn(E, generator=gen, device="cuda")
    d = F.route_backward(cfg, logits, r, dw, ds)
    l = logits.double()
    s, c = torch.sigmoid(l), torch.sigmoid(-l)
    chosen = s.gather(1, r.top_experts)
    g = dw.double()
    if renorm:
        share = chosen / chosen.sum(1, keepdim=True)
        part, size = share * (g - (share * g).sum(1, keepdim=True)), share * (g.abs() + (share * g.abs()).sum(1, keepdim=True))
    else:
        part, size = chosen * g, (chosen * g).abs()
    want = (s * ds.double()).scatter_add(1, r.top_experts, part) * c
    room = (s * ds.double().abs()).scatter_add(1, r.top_experts, size) * c
    assert ((d.double() - want).abs() <= 64 * U * room).all()


@pytest.mark.parametrize("E,dtype", [(128, torch.float32), (127, torch.bfloat16), (256, torch.bfloat16), (512, torch.float32), (1000, torch.bfloat16), (1024, torch.float32)],
                         ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("score,bias,renorm", [("softmax", False, True), ("softmax", False, False), ("sigmoid", False, True), ("sigmoid", True, True),
                                               ("sigmoid", True, False)])
def test_several_rows_per_warp(score, bias, renorm, E, dtype):
    """More rows than the grid has warps: every warp carries its prefetched row, its sums and its shared-memory row on to the next.  All
    values against 64 bits, with d_score_sums and no zero among d_weights; the load figures to what their additions allow."""
    from mok import functional as F
    T = 15013
    logits = logits_of(T, E, dtype, seed=E)
    b = torch.randn(E, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda") * 0.2 if bias else None
    cfg = F.MoKRouterConfig(topk=5, score=score, renormalize=renorm, scale=1.5)
    r = check_forward(cfg, logits, b)
    check_backward(cfg, logits, r)
    # score_sums: a score (its own sum of E / 32 terms a lane and the warp's five steps, 24 more), then positive numbers added: at most
    # 40 rows of a warp (15013 over 148 SMs of three blocks of four warps: 9), 8 warps, 8 blocks a thread of the reduction, 40 more
    _, _, _, sums, _, _ = P.route(logits, 5, score, b, renorm, 1.5)
    rough = (E // 32 + 32 + 40 + 8 + 8 + 40) * U
    assert ((r.score_sums.double() - sums).abs() <= rough * sums).all()


def test_long_batches_of_near_ties():
    """Biased sums a few fp32 steps apart, 120000 rows: every pick is that of the 64-bit sums rounded to 32 bits."""
    from mok import functional as F
    E, K, T = 64, 6, 120000
    gen = torch.Generator(device="cuda").manual_seed(8)
    s = 0.6 + torch.randint(-8, 9, (T, E), generator=gen, device="cuda").double() * 2.0 ** -25
    logits = torch.log(s / (1 - s)).float()
    bias = torch.randint(0, 3, (E,), generator=gen, device="cuda").float() * 2.0 ** -24
    r = F.route(F.MoKRouterConfig(topk=K, score="sigmoid"), logits, bias)
    assert torch.equal(r.top_experts, P.route(logits, K, "sigmoid", bias)[0])


@pytest.mark.parametrize("with_sums", [False, True], ids=["weights", "sums"])
@pytest.mark.parametrize("score,renorm", list(itertools.product(["softmax", "sigmoid"], [True, False])))
def test_a_closed_pick_takes_no_gradient(score, renorm, with_sums):
    """The weight of a closed expert is 0 whatever its logit: a NaN or an infinity in its place among d_router_weights is not looked at."""
    from mok import functional as F
    T, E, K = 64, 40, 6
    logits = logits_of(T, E, torch.float32, seed=11, masked=0.9)
    logits[5] = -torch.inf
    cfg = F.MoKRouterConfig(topk=K, score=score, renormalize=renorm)
    r = F.route(cfg, logits)
    closed = torch.isneginf(logits.gather(1, r.top_experts))
    assert closed.any() and not closed.all()
    gen = torch.Generator(device="cuda").manual_seed(12)
    dw = torch.randn(T, K, generator=gen, device="cuda").masked_fill(closed, 0.0)
    ds = torch.randn(E, generator=gen, device="cuda") if with_sums else None
    want = F.route_backward(cfg, logits, r, dw, ds)
    assert torch.isfinite(want).all()
    for bad in (torch.nan, torch.inf, 1e30):
        assert torch.equal(F.route_backward(cfg, logits, r, dw.masked_fill(closed, bad), ds), want)
