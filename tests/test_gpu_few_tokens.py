"""The layer for a few tokens against a plain implementation in 64 bits."""
import math

import pytest
import torch

from tests import plain_forms as P

pytestmark = pytest.mark.gpu


def make(T, H, I, E, K, *, mx=False, shared=True, total=None, seed=0, std=0.05):
    from mok import ops
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, s=std):
        return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, s, generator=gen)
    x = normal(T, H, s=1.0)
    routed = [normal(E, I, H), normal(E, I, H), normal(E, H, I)]
    if mx:
        routed = [ops.mxfp8_quantize(w, True, False)[:2] for w in routed]
    sh = [normal(I, H), normal(I, H), normal(H, I)] if shared else [None] * 3
    total = total or E
    scores = torch.rand(T, total, generator=gen, device="cuda")
    top = torch.topk(scores, K, dim=1).indices.contiguous()
    w = torch.rand(T, K, generator=gen, device="cuda") + 0.1
    return x, top, w, sh, routed


def check(x, top, w, sh, routed, limit=None, first=0, mx=False, fn=None):
    from mok import _C, functional as F
    y = (fn or F.forward_few_tokens)(x, top, w, *sh, *routed, limit, first_expert=first)
    torch.cuda.synchronize()
    assert _C.check_status() == 0, _C.status_detail()
    assert y.shape == x.shape and y.dtype == torch.bfloat16
    ref, bound = P.few_tokens(x, top, w, None if sh[0] is None else sh, routed, limit, first, mx)
    off = (y.double() - ref).abs()
    assert torch.isfinite(y).all()
    worst = (off / (bound + 1e-30)).max().item()
    assert (off <= bound).all(), f"{worst:.3f} of the bound"
    return y


SIZES = [
    # tokens, hidden, inter, experts, topk
    (1, 256, 128, 1, 1), (1, 1024, 512, 8, 2), (2, 256, 384, 5, 3), (3, 512, 128, 16, 8), (15, 1024, 256, 4, 2),
    (16, 768, 640, 8, 4), (17, 512, 256, 3, 2), (33, 1280, 384, 40, 6), (64, 256, 1408, 6, 1), (100, 512, 128, 2, 2),
    (112, 256, 256, 1, 1), (113, 256, 256, 2, 1), (128, 512, 256, 2, 2), (129, 256, 128, 1, 1), (300, 512, 256, 7, 3),
    (511, 256, 128, 3, 2),
]


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mxfp8"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_against_64_bits(size, mx):
    check(*make(*size, mx=mx, seed=sum(size)), mx=mx)


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mxfp8"])
def test_without_a_shared_expert_and_with_the_clamp(mx):
    args = make(9, 512, 256, 6, 3, mx=mx, shared=False, seed=1, std=0.2)
    check(*args, limit=1.5, mx=mx)
    args = make(20, 512, 256, 6, 3, mx=mx, seed=2, std=0.2)
    check(*args, limit=0.75, mx=mx)


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mxfp8"])
def test_ranks_add_up_and_foreign_routes_give_zeros(mx):
    """Each of four ranks computes its own experts' part; a token none of whose experts is here gets zeros."""
    x, top, w, sh, routed = make(24, 256, 256, 8, 2, mx=mx, total=32, seed=3)
    y = check(x, top, w, [None] * 3, routed, first=8, mx=mx)
    nothing = ((top < 8) | (top >= 16)).all(1)
    assert nothing.any() and not nothing.all()
    assert (y[nothing] == 0).all()
    y = check(x, top + 1000, w, [None] * 3, routed, mx=mx)
    assert (y == 0).all()
    check(x, top + 1000, w, sh, routed, mx=mx)                       # only the shared expert
    y = check(x, torch.full_like(top, -1), w, [None] * 3, routed, mx=mx)
    assert (y == 0).all()


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mxfp8"])
def test_weights_of_zero_and_experts_named_twice(mx):
    x, top, w, sh, routed = make(21, 256, 128, 4, 4, mx=mx, seed=4)
    w[5:] = 0.0                                                      # a padded batch
    w[2, 1] = 0.0
    w[3] *= -1.0
    check(x, top, w, sh, routed, mx=mx)
    top[0, :] = 2                                                    # one expert four times
    top[1, 1] = top[1, 3] = 0
    check(x, top, w, sh, routed, mx=mx)
    top[:] = 3                                                       # 20 routes for two tokens' worth of columns and more
    w = torch.rand_like(w) + 0.1
    check(x, top, w, [None] * 3, routed, mx=mx)
    x, top, w, sh, routed = make(2, 256, 128, 3, 3, mx=mx, seed=5)
    top = torch.zeros(2, 200, dtype=torch.int64, device="cuda")      # 400 routes of two tokens to one expert
    check(x, top, torch.rand(2, 200, device="cuda"), [None] * 3, routed, mx=mx)


def test_weights_of_zero_keep_values_that_are_no_numbers_out():
    """A route without weight reads nothing of its expert: infinities there do not reach the token."""
    x, top, w, sh, routed = make(4, 256, 128, 4, 2, seed=6)
    top[:] = torch.tensor([0, 1], device="cuda")
    top[1, 1] = 3
    w[1, 1] = 0.0
    routed[0][3] = float("inf")
    from mok import functional as F
    y = F.forward_few_tokens(x, top, w, *sh, *routed)
    assert torch.isfinite(y).all()
    w[1, 1] = 1.0
    y = F.forward_few_tokens(x, top, w, *sh, *routed)
    assert y[1].isnan().any() and torch.isfinite(y[[0, 2, 3]]).all()


def test_tokens_that_hold_nan_stay_alone():
    """A column of the product belongs to one token: a NaN in one token's row leaves the others as they are."""
    from mok import functional as F
    x, top, w, sh, routed = make(19, 512, 256, 3, 2, seed=7)
    before = F.forward_few_tokens(x, top, w, *sh, *routed)
    x[4, 100] = float("nan")
    after = F.forward_few_tokens(x, top, w, *sh, *routed)
    assert after[4].isnan().all()
    keep = torch.arange(19, device="cuda") != 4
    assert torch.equal(before[keep], after[keep])


def test_no_tokens():
    from mok import functional as F
    x, top, w, sh, routed = make(1, 256, 128, 2, 1)
    y = F.forward_few_tokens(x[:0], top[:0], w[:0], *sh, *routed)
    assert y.shape == (0, 256)


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mxfp8"])
@pytest.mark.parametrize("size", [(37, 1024, 512, 12, 4), (400, 1024, 256, 5, 3)], ids=["one_unit", "cut_experts"])
def test_two_runs_give_the_same_bits(size, mx):
    """Also where an expert has more tokens than a unit holds: which of its units a token is in must not change."""
    from mok import functional as F
    args = make(*size, mx=mx, seed=8)
    x, top, w, sh, routed = args
    first = F.forward_few_tokens(x, top, w, *sh, *routed)
    for _ in range(20):
        assert torch.equal(first, F.forward_few_tokens(x, top, w, *sh, *routed))


def test_many_routes():
    """More routes than the plan's threads keep in registers (over 4096), with and without cut experts."""
    check(*make(180, 256, 128, 40, 32, seed=13))
    x, top, w, sh, routed = make(511, 256, 128, 16, 12, seed=14)
    check(x, top, w, sh, routed)
    check(x, top, w, [None] * 3, routed, first=3)


def test_two_streams_at_once_and_calls_back_to_back():
    """Calls of different sizes on two streams, many of them in flight: every one has its own work area."""
    from mok import functional as F
    cases = [make(1, 1024, 512, 8, 2, seed=9), make(50, 512, 256, 16, 4, seed=10, mx=True)]
    want = [F.forward_few_tokens(x, t, w, *sh, *r) for x, t, w, sh, r in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(25):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, t, w, sh, r = cases[i]
                got[i].append(F.forward_few_tokens(x, t, w, *sh, *r))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(want[i], y) for y in got[i])


def test_replay_from_two_graphs():
    """Captured twice and replayed on changed inputs, alternately and on two streams."""
    from mok import functional as F
    x, top, w, sh, routed = make(6, 512, 256, 8, 2, seed=11)
    args = (x, top, w, *sh, *routed)
    F.forward_few_tokens(*args)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(F.forward_few_tokens(*args))
        graphs.append(g)
    side = torch.cuda.Stream()
    for scale in (1.0, -0.5, 2.0):
        x.copy_(x * scale)
        top.copy_((top + 1) % 8)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        want = F.forward_few_tokens(*args)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_router_feeds_both_forms_of_the_layer():
    """route -> forward_few_tokens against route -> build_schedule -> forward on the same 512 tokens, taken in pieces."""
    from mok import _C, functional as F
    from tests.gpu_common import init_single_rank_group
    T, H, I, E, K = 512, 512, 256, 8, 2
    x, _, _, sh, routed = make(T, H, I, E, K, seed=12)
    logits = x.float() @ (torch.randn(H, E, device="cuda") * 0.05)
    r = F.route(F.MoKRouterConfig(topk=K), logits)
    cfg = F.MoKConfig(minibatch_size=256, macrobatch_size=T * K * 2 + E * 256, schedule_capacity_multiplier=4.0)
    ws = F.create_workspace(cfg, init_single_rank_group(), device=torch.device("cuda", 0), num_local_tokens=T, hidden_size=H, topk=K)
    sched = F.build_schedule(ws, cfg, r.top_experts, num_local_experts=E)
    whole, _ = F.forward(cfg, ws, sched, x, r.router_weights, *sh, *routed)
    pieces = []
    for lo, hi in ((0, 1), (1, 20), (20, 160), (160, 512)):
        pieces.append(F.forward_few_tokens(x[lo:hi], r.top_experts[lo:hi], r.router_weights[lo:hi], *sh, *routed))
    torch.cuda.synchronize()
    assert _C.check_status() == 0
    ref, bound = P.few_tokens(x, r.top_experts, r.router_weights, sh, routed)
    off = (torch.cat(pieces).double() - ref).abs()
    assert (off <= bound).all()
    # the other form also rounds gate, up and every expert's result to bf16, and both round hidden and y: at most eight roundings of a
    # factor of y, of random sign; four worst cases cover their sum
    assert (whole.double() - torch.cat(pieces).double()).norm() <= 4 * P.U16 * ref.norm()


def test_a_limit_beyond_fp32_limits_nothing():
    from mok import functional as F
    x, e, w, shared, routed = make(5, 256, 128, 4, 2, seed=12)
    want = F.forward_few_tokens(x, e, w, *shared, *routed)
    for limit in (1e300, math.inf, 10 ** 40):
        assert torch.equal(F.forward_few_tokens(x, e, w, *shared, *routed, limit), want)
