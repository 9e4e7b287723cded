"""The router and its gradient against a plain implementation in 64 bits, and the gradient against differences."""
import itertools
import math

import pytest
import torch

from tests import plain_forms as P

pytestmark = pytest.mark.gpu

U = P.U32


def logits_of(T, E, dtype, seed=0, masked=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    l = torch.randn(T, E, generator=gen, device="cuda") * 1.5
    if masked:
        l[torch.rand(T, E, generator=gen, device="cuda") < masked] = -math.inf
    return l.to(dtype)


def check_forward(cfg, logits, bias=None, balance=True):
    from mok import functional as F
    r = F.route(cfg, logits, bias, balance=balance)
    picked, weights, counts, sums, s, _ = P.route(logits, cfg.topk, cfg.score, bias, cfg.renormalize, cfg.scale)
    assert r.top_experts.dtype == torch.int64 and torch.equal(r.top_experts, picked)
    E, K = logits.shape[1], cfg.topk
    # an exp is off by a few roundings (and what its argument's rounding does: |l| < 16 here), sums of E or K by as many
    rel = (E + K + 64) * U
    assert ((r.router_weights.double() - weights).abs() <= rel * weights.abs() + 1e-37).all()
    assert r.router_weights.dtype == torch.float32
    if balance:
        assert r.tokens_per_expert.dtype == torch.int32 and torch.equal(r.tokens_per_expert.long(), counts)
        assert ((r.score_sums.double() - sums).abs() <= (rel + logits.shape[0] * U) * sums + 1e-37).all()
    else:
        assert r.tokens_per_expert is None and r.score_sums is None
    return r


def check_backward(cfg, logits, r, seed=1, with_sums=True):
    from mok import functional as F
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, E = logits.shape
    dw = torch.randn(T, cfg.topk, generator=gen, device="cuda")
    ds = torch.randn(E, generator=gen, device="cuda") * 0.1 if with_sums else None
    d = F.route_backward(cfg, logits, r, dw, ds)
    ref = P.route_bwd(logits, r.top_experts, dw, ds, cfg.score, cfg.renormalize, cfg.scale)
    assert d.dtype == logits.dtype and d.shape == logits.shape and d.is_contiguous()
    # the terms that cancel: s * (ds + the pick's own gradient + their mean), every one off by some (E + K + 64) roundings of itself
    _, _, _, _, s, _ = P.route(logits, cfg.topk, cfg.score, None, cfg.renormalize, cfg.scale)
    chosen = s.gather(1, r.top_experts)
    norm = chosen.sum(1, keepdim=True)
    inv = torch.where(norm > 0, 1.0 / torch.where(norm > 0, norm, 1.0), 0.0) if cfg.renormalize else torch.ones_like(norm)
    each = dw.double().abs() * abs(cfg.scale) * inv
    if cfg.renormalize:
        each = each + (chosen * inv * dw.double().abs() * abs(cfg.scale)).sum(1, keepdim=True) * inv
    terms = torch.zeros_like(s).scatter_add(1, r.top_experts, each) + (ds.double().abs() if ds is not None else 0.0)
    terms = s * (terms + (s * terms).sum(1, keepdim=True))
    bound = 2 * (E + cfg.topk + 64) * U * terms + 1e-37
    if logits.dtype == torch.bfloat16:
        bound = bound + P.U16 * (ref.abs() + bound)
    assert ((d.double() - ref).abs() <= bound).all()
    return d


CONFIGS = list(itertools.product(["softmax", "sigmoid"], [True, False], [torch.float32, torch.bfloat16]))
SIZES = [(1, 1, 1), (1, 256, 8), (3, 8, 8), (7, 33, 5), (64, 60, 6), (130, 128, 4), (257, 129, 7), (100, 260, 8), (50, 512, 8),
         (33, 700, 32), (20, 1024, 16), (1000, 64, 2)]


@pytest.mark.parametrize("score,renorm,dtype", CONFIGS, ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_against_64_bits(size, score, renorm, dtype):
    from mok import functional as F
    T, E, K = size
    cfg = F.MoKRouterConfig(topk=K, score=score, renormalize=renorm, scale=2.5)
    logits = logits_of(T, E, dtype, seed=T + E)
    r = check_forward(cfg, logits)
    check_backward(cfg, logits, r)
    check_backward(cfg, logits, r, with_sums=False)
    check_forward(cfg, logits, balance=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", [(5, 256, 8), (300, 60, 6), (40, 1000, 4)], ids=lambda s: "x".join(map(str, s)))
def test_balancing_bias(size, dtype):
    from mok import functional as F
    T, E, K = size
    cfg = F.MoKRouterConfig(topk=K, score="sigmoid", scale=2.5)
    logits = logits_of(T, E, dtype, seed=5)
    bias = torch.randn(E, device="cuda") * 0.2
    r = check_forward(cfg, logits, bias)
    check_backward(cfg, logits, r)
    assert not torch.equal(r.top_experts, F.route(cfg, logits).top_experts)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
def test_ties_go_to_the_lowest_index(score, bias):
    """Rows of few different values, equal zeros of both signs among them."""
    from mok import functional as F
    if score == "softmax" and bias:
        pytest.skip("a bias goes with sigmoid scores")
    gen = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randint(-1, 2, (500, 96), generator=gen, device="cuda").float()
    logits[:, ::3] *= -1.0                                   # -0.0
    logits[0] = 0.0
    b = torch.randint(0, 2, (96,), generator=gen, device="cuda").float() * 0.25 if bias else None
    cfg = F.MoKRouterConfig(topk=9, score=score)
    r = check_forward(cfg, logits, b)
    if not bias:
        assert torch.equal(r.top_experts[0], torch.arange(9, device="cuda"))


@pytest.mark.parametrize("score,renorm,dtype", CONFIGS, ids=lambda v: str(v).replace("torch.", ""))
def test_closed_experts(score, renorm, dtype):
    """Rows with closed experts, with fewer open ones than topk, with none, with NaN, infinity and the types' extremes."""
    from mok import functional as F
    T, E, K = 40, 72, 6
    logits = logits_of(T, E, dtype, seed=7, masked=0.3)
    logits[3] = -math.inf
    logits[4] = math.nan
    logits[5] = -math.inf
    logits[5, 50] = -3.0
    logits[6] = -math.inf
    logits[6, [70, 2, 9]] = torch.tensor([1.0, 0.5, math.nan], device="cuda").to(dtype)
    logits[8, 11] = math.nan
    logits[9] = torch.finfo(dtype).min
    logits[10, 20] = math.inf
    logits[11] = torch.finfo(dtype).min
    logits[11, 7] = -math.inf
    cfg = F.MoKRouterConfig(topk=K, score=score, renormalize=renorm)
    r = check_forward(cfg, logits)
    assert (r.router_weights[[3, 4]] == 0).all()
    assert torch.equal(r.top_experts[3], torch.arange(K, device="cuda"))
    assert torch.equal(r.top_experts[5], torch.tensor([50, 0, 1, 2, 3, 4], device="cuda"))
    assert torch.isfinite(r.router_weights).all()
    assert (torch.sort(r.top_experts, 1).values.diff(dim=1) > 0).all()          # always K different experts
    d = check_backward(cfg, logits, r)
    assert (d[[3, 4]] == 0).all() and torch.isfinite(d).all()


def test_rows_that_lie_apart_and_odd_addresses():
    from mok import functional as F
    base = logits_of(50, 300, torch.float32, seed=9)
    cfg = F.MoKRouterConfig(topk=4, score="softmax", renormalize=False)
    for view in (base[:, 3:131], base[:, :128], base[:, 1:60], base[1:, 100:228].bfloat16()[:, 1:97]):
        r = check_forward(cfg, view)
        check_backward(cfg, view, r)


@pytest.mark.parametrize("score,renorm", list(itertools.product(["softmax", "sigmoid"], [True, False])))
def test_gradient_against_differences(score, renorm):
    """Central differences of the 64-bit weights around the kernel's own picks."""
    from mok import functional as F
    T, E, K = 4, 12, 3
    cfg = F.MoKRouterConfig(topk=K, score=score, renormalize=renorm, scale=1.5)
    logits = logits_of(T, E, torch.float32, seed=13)
    r = F.route(cfg, logits, balance=True)
    gen = torch.Generator(device="cuda").manual_seed(14)
    dw, ds = torch.randn(T, K, generator=gen, device="cuda"), torch.randn(E, generator=gen, device="cuda")
    d = F.route_backward(cfg, logits, r, dw, ds)
    step = 1e-5

    def loss(l):
        s = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
        w = s.gather(1, r.top_experts)
        w = (w / w.sum(1, keepdim=True) if renorm else w) * 1.5
        return (w * dw.double()).sum() + (s.sum(0) * ds.double()).sum()
    for t, e in itertools.product(range(T), range(E)):
        l = logits.double()
        l[t, e] += step
        up = loss(l)
        l[t, e] -= 2 * step
        slope = (up - loss(l)) / (2 * step)
        # third derivatives of these scores are below 1, gradients of order one: step^2 and the 64-bit differences, and fp32's own error
        assert abs(slope.item() - d[t, e].item()) <= 1e-5


def test_no_tokens():
    from mok import functional as F
    cfg = F.MoKRouterConfig(topk=2)
    logits = torch.zeros(0, 16, device="cuda")
    r = F.route(cfg, logits, balance=True)
    assert r.top_experts.shape == (0, 2) and (r.tokens_per_expert == 0).all() and (r.score_sums == 0).all()
    assert F.route_backward(cfg, logits, r, torch.zeros(0, 2, device="cuda")).shape == (0, 16)


def test_entries_outside_the_experts_have_no_gradient():
    """top_experts that did not come from route: what names no expert is left out, nothing is read for it."""
    from mok import ops
    logits = logits_of(6, 20, torch.float32, seed=15)
    top = torch.tensor([[0, -1], [5, 20], [1 << 40, 3], [7, 7], [2, 3], [-5, 99]], device="cuda")
    dw = torch.ones(6, 2, device="cuda")
    d = ops.route_bwd(logits, top, dw, None, "sigmoid", False, 1.0)
    s = torch.sigmoid(logits.double())
    want = torch.zeros_like(s)
    for t, es in enumerate(top.tolist()):
        for e in es:
            if 0 <= e < 20:
                want[t, e] += s[t, e] * (1 - s[t, e])
    assert ((d.double() - want).abs() <= 64 * U).all()


def test_a_long_batch_and_runs_that_agree():
    from mok import functional as F
    cfg = F.MoKRouterConfig(topk=8)
    logits = logits_of(20000, 256, torch.float32, seed=17)
    r = check_forward(cfg, logits)
    for _ in range(5):
        q = F.route(cfg, logits, balance=True)
        assert all(torch.equal(a, b) for a, b in ((q.top_experts, r.top_experts), (q.router_weights, r.router_weights),
                                                  (q.tokens_per_expert, r.tokens_per_expert), (q.score_sums, r.score_sums)))
    check_backward(cfg, logits, r)


def test_captured_forward_and_backward():
    from mok import functional as F
    cfg = F.MoKRouterConfig(topk=4, score="sigmoid")
    logits, bias = logits_of(100, 64, torch.float32, seed=19), torch.zeros(64, device="cuda")
    dw, ds = torch.randn(100, 4, device="cuda"), torch.randn(64, device="cuda")

    def step():
        r = F.route(cfg, logits, bias, balance=True)
        return r.top_experts, r.router_weights, r.tokens_per_expert, r.score_sums, F.route_backward(cfg, logits, r, dw, ds)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (20, 21):
        logits.copy_(logits_of(100, 64, torch.float32, seed=seed))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_offsets_past_32_bits():
    """More logits than 2^31: the last tokens."""
    from mok import functional as F
    T, E = 2 ** 25 + 5, 64
    logits = torch.empty(T, E, dtype=torch.bfloat16, device="cuda")
    tail = logits_of(9, E, torch.bfloat16, seed=23)
    logits[:-9] = tail[0]
    logits[-9:] = tail
    cfg = F.MoKRouterConfig(topk=3)
    r = F.route(cfg, logits)
    want = F.route(cfg, tail)
    assert torch.equal(r.top_experts[-9:], want.top_experts) and torch.equal(r.router_weights[-9:], want.router_weights)
    dw = torch.zeros(T, 3, device="cuda")
    dw[-9:] = torch.randn(9, 3, device="cuda")
    d = F.route_backward(cfg, logits, r, dw)
    assert torch.equal(d[-9:], F.route_backward(cfg, tail, want, dw[-9:].contiguous())) and (d[:-9] == 0).all()


def test_a_row_whose_order_needs_64_bits():
    """Biased sums that differ by less than a 32-bit sigmoid's error: the order is that of the exact sums."""
    from mok import functional as F
    E, K = 64, 5
    gen = torch.Generator(device="cuda").manual_seed(24)
    logits = torch.randn(300, E, generator=gen, device="cuda")
    s = torch.sigmoid(logits.double())
    bias = torch.zeros(E, device="cuda")
    # every row's logits moved so that all scores lie within 1e-6 of 0.7
    target = 0.7 + (s - 0.5) * 2e-6
    logits = torch.log(target / (1 - target)).float()
    check_forward(F.MoKRouterConfig(topk=K, score="sigmoid"), logits, bias)
    bias = torch.randint(0, 2, (E,), generator=gen, device="cuda").float() * 0.125
    check_forward(F.MoKRouterConfig(topk=K, score="sigmoid"), logits, bias)
    # and fp32 logits that agree in all bits but the last ones
    close = 1.0 + torch.randint(0, 16, (300, E), generator=gen, device="cuda").float() * 2.0 ** -23
    check_forward(F.MoKRouterConfig(topk=K), close)
    check_forward(F.MoKRouterConfig(topk=K), -close)


def test_a_bias_that_is_no_number_comes_last():
    """E = topk takes every expert, whatever the bias holds; picks stay different experts of the row."""
    from mok import functional as F
    for E, K in ((8, 8), (40, 32), (64, 6), (200, 5)):
        logits = logits_of(30, E, torch.float32, seed=E)
        bias = torch.zeros(E, device="cuda")
        bias[0], bias[3], bias[5] = math.nan, -math.inf, math.inf
        r = F.route(F.MoKRouterConfig(topk=K, score="sigmoid"), logits, bias, balance=True)
        order = torch.sigmoid(logits.double()).add(bias.double())
        order[:, 0] = -math.inf
        want = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :K]
        assert torch.equal(r.top_experts, want)
        s = torch.sigmoid(logits.double()).gather(1, want)
        assert ((r.router_weights.double() - s / s.sum(1, keepdim=True)).abs() <= (K + 64) * U).all()
        assert int(r.tokens_per_expert.sum()) == 30 * K
