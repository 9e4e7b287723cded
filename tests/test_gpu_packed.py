"""Activations in 8 bits: packing exact, the backward pass from packed values against 64 bits, and the layer's backward from a
packed context."""
import math

import pytest
import torch

from tests import plain_forms as P

pytestmark = pytest.mark.gpu

SIZES = [(1, 16), (1, 128), (3, 144), (7, 1408), (5, 4096), (33, 112), (130, 256), (1031, 1024), (257, 2000)]


def rows_of(n, c, seed=0, std=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, c, generator=gen, device="cuda") * std
    return (x * torch.exp2(torch.randint(-20, 20, (n, 1), generator=gen, device="cuda").float())).bfloat16()


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_packing_is_exact(size):
    """The whole numbers and the scales are defined to the bit; unpacking rounds their product to bf16 (through one fp32 rounding)."""
    from mok import ops
    x = rows_of(*size, seed=size[1])
    q, scales = ops.pack_rows(x)
    want_q, want_s, values = P.pack(x)
    assert torch.equal(q, want_q) and torch.equal(scales, want_s)
    y = ops.unpack_rows(q, scales)
    assert torch.equal(y, (q.float() * scales.repeat_interleave(128, 1)[:, :size[1]]).bfloat16())
    step = scales.double().repeat_interleave(128, 1)[:, :size[1]]
    off = (y.double() - x.double()).abs()
    assert (off <= step * (0.5 + 127 * 4 * P.U32) + P.U16 * y.double().abs()).all()


def test_every_pair_of_fractions():
    """Every 8-bit fraction of a value against every one of the block's largest, over ten binades: halves go away from zero."""
    from mok import ops
    frac = 1.0 + torch.arange(128, dtype=torch.float64) / 128
    top = frac[:, None, None].expand(128, 10, 128)
    v = (frac[None, None, :] * torch.exp2(-torch.arange(10, dtype=torch.float64))[None, :, None]).expand(128, 10, 128)
    x = torch.minimum(v, top).clone()
    x[..., 1::2] *= -1.0
    x[..., 127] = top[..., 0]
    x = x.reshape(-1, 128).bfloat16().cuda()
    assert torch.equal(x.double().abs().amax(1), top[..., 0].reshape(-1).cuda())
    q, scales = ops.pack_rows(x)
    want_q, want_s, _ = P.pack(x)
    assert torch.equal(q, want_q) and torch.equal(scales, want_s)
    assert ((x.double().abs() * 254 / top[..., :1].reshape(-1, 1).cuda()) % 2 == 1).any()        # there are halves


def test_extremes():
    from mok import ops
    big = torch.finfo(torch.bfloat16).max
    x = torch.zeros(10, 256, dtype=torch.bfloat16, device="cuda")
    x[1, 3] = big
    x[1, 4] = -big
    x[1, 200] = big / 2
    x[2, :128] = 2.0 ** -130
    x[3, 7] = 2.0 ** -110
    x[3, 8] = -(2.0 ** -117)
    x[4, 5] = math.inf
    x[5, 5] = math.nan
    x[6, 130] = -math.inf
    x[7] = -0.0
    x[8] = torch.finfo(torch.bfloat16).tiny
    x[9] = 3.0
    q, scales = ops.pack_rows(x)
    want_q, want_s, _ = P.pack(x)
    assert torch.equal(q, want_q)
    assert torch.equal(scales.nan_to_num(-1.0), want_s.nan_to_num(-1.0))
    y = ops.unpack_rows(q, scales)
    assert y[4, :128].isnan().all() and y[5, :128].isnan().all() and y[6, 128:].isnan().all()      # a fault stays visible, in its block
    assert (y[4:6, 128:] == 0).all() and (y[6, :128] == 0).all()
    assert y[1, 3] == big and y[1, 4] == -big and (y[9] == 3.0).all()
    assert (y[[0, 2, 7, 8]] == 0).all()


@pytest.mark.parametrize("limit", [None, 1.25], ids=["free", "clamped"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_swiglu_backward(size, limit):
    from mok import ops
    n, c = size
    gen = torch.Generator(device="cuda").manual_seed(n + c)
    gate, up, dh = (torch.randn(n, c, generator=gen, device="cuda").mul(2.0).bfloat16() for _ in range(3))
    gate[0, 0] = -90.0                                    # exp overflows
    gate[-1, -1] = 90.0
    w = torch.rand(n, generator=gen, device="cuda") + 0.01
    w[::5] = 0.0
    w[1::7] = -1.0
    gp, upk = ops.pack_rows(gate), ops.pack_rows(up)
    g, u = P.pack(gate)[2].float().double(), P.pack(up)[2].float().double()       # one fp32 rounding of the product
    for row_scale in (w, None):
        got = ops.swiglu_bwd_packed(*gp, *upk, dh, limit, row_scale)
        want = P.swiglu_bwd(g, u, dh.double(), limit, row_scale)
        # silu and its derivative in fp32: some 16 roundings of their own terms (silu' = sig + g sig (1 - sig), both terms counted), and
        # an exp whose argument of up to 90 is rounded: 90 roundings
        gc = g if limit is None else g.clamp(max=limit)
        uc = u if limit is None else u.clamp(-limit, limit)
        sigc = torch.sigmoid(gc)
        terms = (sigc + (gc * sigc).abs() * (1 + sigc)) * uc.abs() * dh.double().abs()
        rough = 128 * P.U32
        # sig is below fp32's smallest normal number for gates under -87.3 and may be lost there: 2^-126, times what multiplies it
        lost = 2.0 ** -126 * (1 + (2 + gc.abs()) * (1 + uc.abs()) * dh.double().abs().clamp_min(1.0))
        for name, a, b, t in (("d_gate", got[0], want[0], terms), ("d_up", got[1], want[1], want[1].abs()), ("hidden", got[2], want[2], want[2].abs())):
            assert ((a.double() - b).abs() <= rough * t + P.U16 * (b.abs() + rough * t) + lost).all(), name
        inv = torch.ones_like(want[3]) if row_scale is None else torch.where(w.double() > 0, 1 / w.double(), 0.0)
        total = (dh.double() * want[2]).abs().sum(1) * inv
        assert ((got[3].double() - want[3]).abs() <= (c + 128) * P.U32 * total + lost.sum(1) * (1 + inv)).all()


@pytest.mark.parametrize("size", [(5, 131072), (11, 16400), (3, 32784), (2049, 16), (257, 4080)], ids=lambda s: "x".join(map(str, s)))
def test_swiglu_backward_wide_and_narrow_rows(size):
    """Rows wider than a block's shared memory holds eight of, and units that straddle 128 values; each row's results are the row's alone."""
    from mok import ops
    n, c = size
    gen = torch.Generator(device="cuda").manual_seed(n * c)
    gate, up, dh = (torch.randn(n, c, generator=gen, device="cuda").bfloat16() for _ in range(3))
    gp, upk = ops.pack_rows(gate), ops.pack_rows(up)
    w = torch.rand(n, generator=gen, device="cuda") + 0.5
    got = ops.swiglu_bwd_packed(*gp, *upk, dh, None, w)
    g, u, d = P.pack(gate)[2].double(), P.pack(up)[2].double(), dh.double()
    want = P.swiglu_bwd(g, u, d, None, w)
    sig = torch.sigmoid(g)
    terms = ((sig + (g * sig).abs() * (1 + sig)) * u.abs() * d.abs(), want[1].abs(), want[2].abs())       # as in test_swiglu_backward
    for a, b, e in zip(got[:3], want[:3], terms):
        assert ((a.double() - b).abs() <= 128 * P.U32 * e + P.U16 * (b.abs() + 128 * P.U32 * e)).all()
    total = (dh.double() * want[2]).abs().sum(1) / w.double()
    assert ((got[3].double() - want[3]).abs() <= (c + 128) * P.U32 * total).all()
    for row in (0, n // 2, n - 1):
        one = [t[row:row + 1].contiguous() for t in (*gp, *upk, dh)]
        alone = ops.swiglu_bwd_packed(*one, None, w[row:row + 1].contiguous())
        assert all(torch.equal(a[0], b[row]) for a, b in zip(alone, got))


def test_gradient_against_differences():
    from mok import ops
    gen = torch.Generator(device="cuda").manual_seed(2)
    gate, up = (torch.randn(2, 16, generator=gen, device="cuda").bfloat16() for _ in range(2))
    dh = torch.ones(2, 16, dtype=torch.bfloat16, device="cuda")
    got = ops.swiglu_bwd_packed(*ops.pack_rows(gate), *ops.pack_rows(up), dh)
    g, u = P.pack(gate)[2], P.pack(up)[2]
    step = 1e-6

    def h(a, b):
        return a * torch.sigmoid(a) * b
    for out, slope in ((got[0], (h(g + step, u) - h(g - step, u)) / (2 * step)), (got[1], (h(g, u + step) - h(g, u - step)) / (2 * step))):
        assert ((out.double() - slope).abs() <= 2 * P.U16 * slope.abs() + 1e-6).all()


def test_a_fault_in_gate_or_up_stays_visible():
    from mok import ops
    gate, up, dh = (torch.ones(3, 128, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    gate[0, 3] = math.nan
    up[1, 4] = math.inf
    for limit in (None, 0.5):
        d_gate, d_up, hidden, grad = ops.swiglu_bwd_packed(*ops.pack_rows(gate), *ops.pack_rows(up), dh, limit)
        assert hidden[:2].isnan().all() and grad[:2].isnan().all() and torch.isfinite(hidden[2]).all() and torch.isfinite(grad[2])
        assert d_gate[0].isnan().all()
        # the other factor is 1.0: beyond a limit of 0.5 its gradient is zero whatever it is multiplied by
        for other in (d_gate[1], d_up[0]):
            assert other.isnan().all() if limit is None else (other == 0).all()


def test_rows_behind_the_last_stay_as_they_were():
    """With a row count on the device nothing behind it is read or written; counts beyond the tensor and below zero are held."""
    from mok import _C
    x, u, dh = rows_of(40, 272, seed=4), rows_of(40, 272, seed=5), rows_of(40, 272, seed=6, std=1e-3)
    full_q, full_s = _C.pack_rows(x)
    up_q, up_s = _C.pack_rows(u)
    full_y = _C.unpack_rows(full_q, full_s)
    full_b = _C.swiglu_bwd_packed(full_q, full_s, up_q, up_s, dh)
    lib, p, st = _C.lib, _C._p, _C._stream
    for count in (0, 1, 17, 40, 1000, -3):
        num = torch.tensor([count], dtype=torch.int32, device="cuda")
        n = min(max(count, 0), 40)
        q, s = torch.full_like(full_q, 77), torch.full_like(full_s, -5.0)
        _C._ck(lib.mokb_pack_rows(p(x), p(q), p(s), p(num), 40, 272, st()))
        assert torch.equal(q[:n], full_q[:n]) and (q[n:] == 77).all() and torch.equal(s[:n], full_s[:n]) and (s[n:] == -5.0).all()
        y = torch.full_like(full_y, 9.0)
        _C._ck(lib.mokb_unpack_rows(p(full_q), p(full_s), p(y), p(num), 40, 272, st()))
        assert torch.equal(y[:n], full_y[:n]) and (y[n:] == 9.0).all()
        outs = [torch.full_like(t, 9.0) for t in full_b]
        _C._ck(lib.mokb_swiglu_bwd_packed(p(full_q), p(full_s), p(up_q), p(up_s), p(dh), *(p(t) for t in outs[:3]), None, p(outs[3]), p(num),
                                          40, 272, 0, 0.0, st()))
        for got, want in zip(outs, full_b):
            assert torch.equal(got[:n], want[:n]) and (got[n:] == 9.0).all()


def test_offsets_past_32_bits():
    """More values than 2^31: the last rows of all three."""
    from mok import ops
    n, c = 2 ** 20 + 3, 2048
    tail = rows_of(5, c, seed=31)
    x = torch.zeros(n, c, dtype=torch.bfloat16, device="cuda")
    x[-5:] = tail
    q, s = ops.pack_rows(x)
    tq, ts = ops.pack_rows(tail)
    assert torch.equal(q[-5:], tq) and torch.equal(s[-5:], ts) and int(q[:-5].abs().max()) == 0
    del x
    assert torch.equal(ops.unpack_rows(q, s)[-5:], ops.unpack_rows(tq, ts))
    dh = torch.ones(n, c, dtype=torch.bfloat16, device="cuda")
    got, want = ops.swiglu_bwd_packed(q, s, q, s, dh), ops.swiglu_bwd_packed(tq, ts, tq, ts, dh[:5])
    assert all(torch.equal(a[-5:], b) for a, b in zip(got, want))


def test_no_rows():
    from mok import ops
    q, s = ops.pack_rows(torch.zeros(0, 256, dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (0, 256) and s.shape == (0, 2) and ops.unpack_rows(q, s).shape == (0, 256)


# ---------------------------------------------------------------------------------------------------------------- the layer
def layer(T, H, I, E, K, macro=None, seed=21, limit=None):
    from mok import functional as F
    from oracle import mok_oracle as O
    from tests.gpu_common import init_single_rank_group, to_dev
    inp = to_dev(O.make_inputs(R=1, T=T, H=H, I=I, E=E, K=K, seed=seed, routing="router")[0])
    cfg = F.MoKConfig(minibatch_size=256, macrobatch_size=macro or (T * K + E * 256 + 255) // 256 * 256, schedule_capacity_multiplier=4.0,
                      all_gather_top_experts_chunk_bytes=1024)
    ws = F.create_workspace(cfg, init_single_rank_group(), device=torch.device("cuda", 0), num_local_tokens=T, hidden_size=H, topk=K)
    sched = F.build_schedule(ws, cfg, inp.top_experts, num_local_experts=E)
    shared = (inp.w_shared_gate, inp.w_shared_up, inp.w_shared_down)
    routed = (inp.w_routed_gate, inp.w_routed_up, inp.w_routed_down)
    _, ctx = F.forward(cfg, ws, sched, inp.x, inp.router_weights, *shared, *routed, limit)

    def backward(c):
        return F.backward(cfg, ws, sched, c, inp.grad_output, inp.x, inp.router_weights, *shared, *routed, limit)
    return F, cfg, ws, sched, inp, ctx, backward


NAMES = ("d_x", "d_router_weights", "d_routed_gate", "d_routed_up", "d_routed_down", "d_shared_gate", "d_shared_up", "d_shared_down")


@pytest.mark.parametrize("limit", [None, 1.0], ids=["free", "clamped"])
@pytest.mark.parametrize("case", [(512, 512, 256, 8, 2, None), (768, 256, 384, 5, 3, None), (1024, 512, 256, 6, 2, 1024)],
                         ids=["512", "768_odd", "macrobatches"])
def test_backward_from_a_packed_context(case, limit):
    """Against the same backward pass of the context that the packed values stand for: x, gate and up unpacked, hidden from them."""
    from mok import _C, ops
    F, cfg, ws, sched, inp, ctx, backward = layer(*case, limit=limit)
    packed = F.pack_context(sched, ctx)
    n = min(int(sched.num_tokens.item()), cfg.macrobatch_size)
    before = [t.clone() for pair in (packed.x_routed, packed.gate_routed, packed.up_routed, packed.gate_shared, packed.up_shared) for t in pair]
    got = backward(packed)
    torch.cuda.synchronize()
    assert _C.check_status() == 0, _C.status_detail()
    after = [t for pair in (packed.x_routed, packed.gate_routed, packed.up_routed, packed.gate_shared, packed.up_shared) for t in pair]
    for i, (a, b) in enumerate(zip(before, after)):
        rows = n if i < 6 else a.shape[0]
        assert torch.equal(a[:rows], b[:rows])            # the context is left as it is

    def unpacked(pair, like):
        out = like.clone()
        rows = n if like.shape[0] == cfg.macrobatch_size else like.shape[0]
        out[:rows] = ops.unpack_rows(*pair)[:rows]
        return out
    g, u = unpacked(packed.gate_routed, ctx.gate_routed), unpacked(packed.up_routed, ctx.up_routed)
    gs, us = unpacked(packed.gate_shared, ctx.gate_shared), unpacked(packed.up_shared, ctx.up_shared)
    stand_in = F.MoKForwardContext(x_routed=unpacked(packed.x_routed, ctx.x_routed), gate_shared=gs, gate_routed=g, up_shared=us, up_routed=u,
                                   hidden_shared=_C.swiglu_fwd(gs, us, limit), hidden_routed=_C.swiglu_fwd(g, u, limit))
    want = backward(stand_in)
    torch.cuda.synchronize()
    # the stand-in rounds gate and up to bf16 (and hidden from those): three roundings of each factor, and with a clamp the few values
    # that a rounding moves across it
    for name, a, b in zip(NAMES, got, want):
        rel = ((a.double() - b.double()).norm() / b.double().norm()).item()
        assert rel <= (8 if limit is None else 16) * P.U16, (name, rel)


def test_packed_context_is_near_the_whole_one():
    """Gradients from 8 bits against those from bf16: x, gate and up are off by half a step of 1/127 of their block's largest value,
    about 0.7 % of a value of ordinary size, in each factor."""
    from mok import _C
    F, cfg, ws, sched, inp, ctx, backward = layer(512, 512, 256, 8, 2)
    packed = F.pack_context(sched, ctx)
    got, want = backward(packed), backward(ctx)
    torch.cuda.synchronize()
    assert _C.check_status() == 0
    for name, a, b in zip(NAMES, got, want):
        rel = ((a.double() - b.double()).norm() / b.double().norm()).item()
        assert rel <= 0.03, (name, rel)
    size = sum(t.nbytes for pair in (packed.x_routed, packed.gate_routed, packed.up_routed, packed.gate_shared, packed.up_shared) for t in pair)
    whole = sum(t.nbytes for t in (ctx.x_routed, ctx.gate_routed, ctx.up_routed, ctx.hidden_routed, ctx.gate_shared, ctx.up_shared, ctx.hidden_shared))
    assert size < 0.45 * whole


def test_a_training_step_with_router_and_packed_context_replays_from_a_graph():
    """route -> schedule -> forward -> pack -> backward -> route_backward, captured; eager results bit for bit on changed inputs."""
    from mok import _C
    F, cfg, ws, sched, inp, ctx, _ = layer(512, 512, 256, 8, 2)
    rcfg = F.MoKRouterConfig(topk=2)
    shared = (inp.w_shared_gate, inp.w_shared_up, inp.w_shared_down)
    routed = (inp.w_routed_gate, inp.w_routed_up, inp.w_routed_down)
    x, gy = inp.x.clone(), inp.grad_output.clone()
    wr = torch.randn(512, 8, device="cuda") * 0.05
    logits = torch.empty(512, 8, device="cuda")

    def step():
        torch.mm(x.float(), wr, out=logits)
        r = F.route(rcfg, logits, balance=True)
        s = F.build_schedule(ws, cfg, r.top_experts, num_local_experts=8)
        y, c = F.forward(cfg, ws, s, x, r.router_weights, *shared, *routed)
        p = F.pack_context(s, c)
        del c
        grads = F.backward(cfg, ws, s, p, gy, x, r.router_weights, *shared, *routed)
        return (y, *grads, F.route_backward(rcfg, logits, r, grads[1], r.score_sums * 1e-3), r.tokens_per_expert)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for scale in (1.0, 0.5):
        x.copy_(inp.x * scale)
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = step()
        torch.cuda.synchronize()
        assert _C.check_status() == 0
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), i
