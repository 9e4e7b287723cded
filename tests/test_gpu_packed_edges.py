"""The backward pass of SwiGLU (whole, packed and quantising) at weights where 1 / w leaves fp32's range, at rows without a weight, and
the packed form's arithmetic against the whole one's."""
import math

import pytest
import torch

from tests import plain_forms as P

pytestmark = pytest.mark.gpu


def whole_numbers(rows, cols, seed):
    """bf16 values that packing holds exactly: whole numbers up to 127 times a power of two per block, 127 in every block."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randint(-127, 128, (rows, cols // 128, 128), generator=gen, device="cuda").float()
    v[..., 0] = 127.0
    v *= torch.exp2(torch.randint(-9, 1, (rows, cols // 128, 1), generator=gen, device="cuda").float())
    return v.view(rows, cols).bfloat16()


TINY = [1e-45, 1e-42, 1e-39, 2.0 ** -128, 2.0 ** -127, 2.0 ** -126, 1e-30, 0.5]


def rows_with_zeros(n, c, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    gate, up, dh = (torch.randn(n, c, generator=gen, device="cuda").bfloat16() for _ in range(3))
    gate[:, 1::5] = 0.0
    dh[:, 2::7] = 0.0
    return gate, up, dh


def check_row_gradient(got, gate, up, dh, w):
    """sum(d_hidden * hidden) / w of d_hidden that is as small as w: c products and a sum in fp32 of terms that the rows' weights bring
    back to ordinary size, a quotient, and silu's own roundings (as test_gpu_packed.py counts them)."""
    c = gate.shape[1]
    terms = dh.double() * (gate * torch.sigmoid(gate) * up)
    want = torch.where(w > 0, terms.sum(1) / torch.where(w > 0, w, 1.0).double(), 0.0)
    room = torch.where(w > 0, terms.abs().sum(1) / torch.where(w > 0, w, 1.0).double(), 0.0)
    assert torch.isfinite(got).all(), got
    assert ((got.double() - want).abs() <= (c + 128) * P.U32 * room).all(), (got, want)


def scaled(dh, w):
    """d_hidden of rows scaled by their weights: bf16, exact where the product is a normal number."""
    return (dh.double() * w.double()[:, None]).bfloat16()


def test_row_gradient_of_tiny_weights_packed():
    from mok import ops
    w = torch.tensor(TINY, device="cuda")
    gate, up, dh = rows_with_zeros(len(TINY), 512)
    dh = scaled(dh, w)
    gp, upk = ops.pack_rows(gate), ops.pack_rows(up)
    got = ops.swiglu_bwd_packed(*gp, *upk, dh, None, w)[3]
    check_row_gradient(got, P.pack(gate)[2], P.pack(up)[2], dh, w)


def test_row_gradient_of_tiny_weights_whole():
    from mok import _C
    w = torch.tensor(TINY, device="cuda")
    gate, up, dh = rows_with_zeros(len(TINY), 512)
    dh = scaled(dh, w)
    got = _C.swiglu_bwd(gate, up, dh, None, w, True)[2]
    check_row_gradient(got, gate.double(), up.double(), dh, w)


@pytest.mark.parametrize("precision", ["bf16", "packed", "mxfp8"])
def test_router_gradients_of_the_layer_at_tiny_weights(precision):
    """Routes whose weight is positive but below 2^-128 (a softmax that is not renormalised has such): their scaled rows underflow, and
    the router's gradient stays a number.  Every other route's gradients are as in a run without them."""
    from mok import _C, functional as F, ops
    from oracle import mok_oracle as O
    from tests.gpu_common import init_single_rank_group, to_dev
    T, H, I, E, K = 512, 512, 256, 8, 2
    inp = to_dev(O.make_inputs(R=1, T=T, H=H, I=I, E=E, K=K, seed=33, routing="router")[0])
    cfg = F.MoKConfig(minibatch_size=256, macrobatch_size=(T * K + E * 256 + 255) // 256 * 256, schedule_capacity_multiplier=4.0)
    ws = F.create_workspace(cfg, init_single_rank_group(), device=torch.device("cuda", 0), num_local_tokens=T, hidden_size=H, topk=K)
    sched = F.build_schedule(ws, cfg, inp.top_experts, num_local_experts=E)
    shared = (inp.w_shared_gate, inp.w_shared_up, inp.w_shared_down)
    routed = bwd = (inp.w_routed_gate, inp.w_routed_up, inp.w_routed_down)
    if precision == "mxfp8":
        q = [ops.mxfp8_quantize(t, True, True) for t in routed]
        routed = tuple(t[:2] for t in q)
        bwd = (q[0], q[1], q[2][2:])

    def gradients(weights):
        _, ctx = F.forward(cfg, ws, sched, inp.x, weights, *shared, *routed)
        if precision == "packed":
            ctx = F.pack_context(sched, ctx)
        grads = F.backward(cfg, ws, sched, ctx, inp.grad_output, inp.x, weights, *shared, *bwd)
        torch.cuda.synchronize()
        assert _C.check_status() == 0
        return grads
    plain = gradients(inp.router_weights)
    weights = inp.router_weights.clone()
    weights[::3, 1] = 1e-42
    weights[1::3, 0] = 1e-39
    d_x, d_w = gradients(weights)[:2]
    assert torch.isfinite(d_w).all() and torch.isfinite(d_x).all()
    same = weights == inp.router_weights
    assert torch.equal(d_w[same], plain[1][same])


def test_a_row_without_a_weight_has_no_row_gradient():
    """0 where row_scale is not positive (or not a number), whatever the row holds: a block that came back as NaN, a product past
    fp32's range, an infinite d_hidden."""
    from mok import ops
    c = 256
    gate, up, dh = (torch.ones(8, c, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    gate[0, 3] = math.nan
    up[1, 200] = -math.inf
    gate[2], up[2] = 3e38, 3e38
    dh[3, 5] = math.inf
    dh[4, 6] = math.nan
    w = torch.tensor([0.0, -0.0, 0.0, -1.0, 0.0, math.nan, -math.inf, 1.0], device="cuda")
    for limit in (None, 7.0):
        got = ops.swiglu_bwd_packed(*ops.pack_rows(gate), *ops.pack_rows(up), dh, limit, w)[3]
        assert (got[:7] == 0).all(), got
        assert torch.isfinite(got[7]) and got[7] > 0


@pytest.mark.parametrize("limit", [None, 7.0, 0.25], ids=["free", "7", "quarter"])
def test_packed_gradients_are_the_whole_forms_to_the_bit(limit):
    """Of gate and up that packing holds exactly, d_gate and d_up are mokb_swiglu_bwd's: the same operations on the same numbers, none
    of them in fewer bits."""
    from mok import _C, ops
    n, c = 2048, 1024
    gate, up = whole_numbers(n, c, 3), whole_numbers(n, c, 4)
    dh = torch.randn(n, c, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").bfloat16()
    gp, upk = ops.pack_rows(gate), ops.pack_rows(up)
    assert torch.equal(ops.unpack_rows(*gp), gate) and torch.equal(ops.unpack_rows(*upk), up)
    got = ops.swiglu_bwd_packed(*gp, *upk, dh, limit)
    want = _C.swiglu_bwd(gate, up, dh, limit)
    assert torch.equal(got[0], want[0]), int((got[0] != want[0]).sum())
    assert torch.equal(got[1], want[1]), int((got[1] != want[1]).sum())
