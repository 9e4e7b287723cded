"""The layer's backward operator from a packed context where rows come from and go to other ranks (every "peer" a buffer of its own on
this GPU, each rank's calls made in turn: the kernels never wait on one another), and its schema and fake kernel."""
import pytest
import torch

from oracle import mok_oracle as O
from tests import plain_forms as P
from tests.test_gpu_local_peers import make_routes

pytestmark = pytest.mark.gpu


class Ranks:
    """R ranks' inputs, weights and buffers; rank q holds the experts [q * E_l, (q + 1) * E_l)."""

    def __init__(self, R, T, K, H, I, E_l, MB, limit, seed):
        self.R, self.T, self.K, self.H, self.I, self.E_l, self.MB, self.limit = R, T, K, H, I, E_l, MB, limit
        routes = make_routes(R, T, K, E_l, seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        bf = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).bfloat16()
        self.x, self.dy = ([bf(T, H) for _ in range(R)] for _ in range(2))
        self.w = [torch.rand(T, K, generator=g, device="cuda") + 0.05 for _ in range(R)]
        self.weights = [[bf(I, H, std=0.05), bf(E_l, I, H, std=0.05), bf(I, H, std=0.05), bf(E_l, I, H, std=0.05), bf(H, I, std=0.05),
                         bf(E_l, H, I, std=0.05)] for _ in range(R)]      # shared and routed gate, up, down
        C = (T * K * R + E_l * 256 + 255) // 256 * 256
        self.schedules = [[torch.from_numpy(a).cuda() for a in O.schedule(routes, E_l, C, q)] for q in range(R)]
        self.routes = routes

    def buffers(self):
        return ([torch.zeros(self.T * self.K, self.H, dtype=torch.bfloat16, device="cuda") for _ in range(self.R)],
                [torch.full((self.T, self.K), -7.0, device="cuda") for _ in range(self.R)])

    def context(self, q):
        from mok import ops
        sg, rg, su, ru, _, _ = self.weights[q]
        return ops.recompute_forward_context_bf16(self.x[q], ptrs(self.x), sg, rg, su, ru, *self.schedules[q], self.K, self.limit, 16,
                                                  self.MB, 256)

    def arguments(self, q, context, d_x, d_w):
        return (self.dy[q], ptrs(self.dy), d_x[q], ptrs(d_x), self.w[q], ptrs(self.w), d_w[q], ptrs(d_w), *self.weights[q], *context,
                self.x[q], ptrs(self.x), *self.schedules[q], self.K, self.limit, 16, self.MB, 256)


def ptrs(tensors):
    return [t.data_ptr() for t in tensors]


def pack(context, num_tokens):
    """x_routed, gate_routed, up_routed, gate_shared, up_shared in 8 bits, in the operator's order, and what they stand for."""
    from mok import _C, ops
    x, gs, gr, us, ur = context[:5]
    pairs = [ops.pack_rows(x, num_tokens), ops.pack_rows(gr, num_tokens), ops.pack_rows(ur, num_tokens), ops.pack_rows(gs), ops.pack_rows(us)]
    return [t for pair in pairs for t in pair], [ops.unpack_rows(*pair) for pair in pairs]


@pytest.mark.parametrize("R,T,K,H,I,E_l,MB,limit", [(2, 512, 2, 512, 256, 3, 4096, None), (4, 512, 4, 256, 384, 2, 8704, 1.0),
                                                    (3, 768, 2, 256, 256, 2, 1024, None)], ids=["two", "four_clamped", "three_macrobatches"])
def test_backward_over_local_peers(R, T, K, H, I, E_l, MB, limit):
    """Every rank's gradients, and the rows and router-weight gradients that all ranks sent home, from the packed context against the same
    call with the context that the packed values stand for (rounded to bf16: three roundings of each factor, and with a clamp the few
    values that a rounding moves across it: test_gpu_packed.py's bounds)."""
    from mok import _C, ops
    ranks = Ranks(R, T, K, H, I, E_l, MB, limit, seed=130 + R)
    got_home, want_home = ranks.buffers(), ranks.buffers()
    tol = (8 if limit is None else 16) * P.U16
    remote = 0

    def near(name, a, b):
        rel = ((a.double() - b.double()).norm() / b.double().norm()).item()
        assert rel <= tol, (name, rel)
    for q in range(R):
        peer = ranks.schedules[q][0][:int(ranks.schedules[q][2])]
        remote += int(((peer >= 0) & (peer != q)).sum())
        context = ranks.context(q)
        n = min(int(ranks.schedules[q][2]), MB)
        packed, (x, gr, ur, gs, us) = pack(context, ranks.schedules[q][2])
        kept = [t.clone() for t in packed]
        got = ops.dispatch_mlp_swiglu_combine_bwd_bf16_packed(*ranks.arguments(q, packed, *got_home))
        torch.cuda.synchronize()
        assert _C.check_status() == 0, _C.status_detail()
        for i, (a, b) in enumerate(zip(kept, packed)):          # the context is left as it is (rows behind the last hold nothing)
            rows = n if i < 6 else T
            assert torch.equal(a[:rows].nan_to_num(), b[:rows].nan_to_num())
        stand_in = []
        for whole, back in ((context[0], x), (context[1], gs), (context[2], gr), (context[3], us), (context[4], ur)):
            t = whole.clone()
            rows = T if whole is context[1] or whole is context[3] else n
            t[:rows] = back[:rows]
            stand_in.append(t)
        stand_in += [_C.swiglu_fwd(stand_in[1], stand_in[3], limit), _C.swiglu_fwd(stand_in[2], stand_in[4], limit)]
        want = ops.dispatch_mlp_swiglu_combine_bwd_bf16(*ranks.arguments(q, stand_in, *want_home))
        torch.cuda.synchronize()
        assert _C.check_status() == 0, _C.status_detail()
        near("d_x_shared", got[0], want[0])
        for i in range(-6, 0):
            near(f"weight gradient {i}", got[i], want[i])
    assert remote > 0
    for r in range(R):
        near(f"rank {r}'s rows", got_home[0][r], want_home[0][r])
        near(f"rank {r}'s router weights", got_home[1][r], want_home[1][r])
        assert (got_home[1][r] != -7.0).all()                   # every route came home


def test_schema_and_fake_kernel():
    """Under SchemaCheckMode the operator mutates what its schema says and nothing else; its fake kernel gives its outputs' shapes and
    types.  (opcheck copies its arguments, whose addresses would then not be the pointer lists'.)"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch._subclasses.schema_check_mode import SchemaCheckMode
    from mok import _C, ops
    ranks = Ranks(2, 512, 2, 256, 256, 2, 2560, None, seed=140)
    home = ranks.buffers()
    packed, _ = pack(ranks.context(0), ranks.schedules[0][2])
    args = ranks.arguments(0, packed, *home)
    op = torch.ops.mok.dispatch_mlp_swiglu_combine_bwd_bf16_packed
    with SchemaCheckMode():
        outs = op(*args)
    torch.cuda.synchronize()
    assert _C.check_status() == 0
    with FakeTensorMode() as mode:
        fakes = op(*(mode.from_tensor(a) if isinstance(a, torch.Tensor) else a for a in args))
    assert len(outs) == len(fakes)
    for a, b in zip(outs, fakes):
        assert a.shape == b.shape and a.dtype == b.dtype and a.device == b.device and a.stride() == b.stride()
