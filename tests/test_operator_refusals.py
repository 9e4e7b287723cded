"""What the operators around the layer refuse, before any device work: run on the CPU (a tensor that is not on a GPU is itself refused,
after its type and shape), and the library's own checks, which see sizes and addresses but read nothing."""
import ctypes

import pytest
import torch

BF, F32, I64, I8 = torch.bfloat16, torch.float32, torch.int64, torch.int8


def test_router_arguments():
    from mok import functional as F, ops
    l = torch.zeros(4, 16)
    ok = dict(bias=None, topk=2, score="softmax", renormalize=True, scale=1.0, balance=False)
    def call(logits=l, **kw):
        a = {**ok, **kw}
        return ops.route(logits, a["bias"], a["topk"], a["score"], a["renormalize"], a["scale"], a["balance"])
    with pytest.raises(ValueError, match="CUDA tensor"):
        call()
    for kw, error, why in (
            (dict(topk=0), ValueError, "topk"), (dict(topk=33), ValueError, "topk"), (dict(topk=17), ValueError, "num_experts"),
            (dict(score="relu"), ValueError, "score"), (dict(scale=float("nan")), ValueError, "scale"), (dict(scale=-float("inf")), ValueError, "scale"),
            (dict(scale=1e39), ValueError, "scale"),
            (dict(logits=torch.zeros(4, 1025)), ValueError, "num_experts"), (dict(logits=torch.zeros(16)), ValueError, "shape"),
            (dict(logits=torch.zeros(4, 16, dtype=torch.float16)), TypeError, "dtype"), (dict(logits=l.double()), TypeError, "dtype")):
        with pytest.raises(error, match=why):
            call(**kw)
    with pytest.raises(ValueError, match="top_experts"):
        ops.route_bwd(l, torch.zeros(4, dtype=I64), torch.zeros(4, 2), None, "softmax", True, 1.0)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.route_bwd(l, torch.zeros(4, 2, dtype=I64), torch.zeros(4, 2), None, "softmax", True, 1.0)
    with pytest.raises(TypeError, match="MoKRouterConfig"):
        F.route(F.MoKConfig(), l)
    with pytest.raises(TypeError, match="MoKRouting"):
        F.route_backward(F.MoKRouterConfig(topk=2), l, None, torch.zeros(4, 2))


def few(T=4, H=256, I=128, E=2, K=2, **kw):
    from mok import functional as F
    a = dict(x=torch.zeros(T, H, dtype=BF), top=torch.zeros(T, K, dtype=I64), w=torch.zeros(T, K), sg=torch.zeros(I, H, dtype=BF),
             su=torch.zeros(I, H, dtype=BF), sd=torch.zeros(H, I, dtype=BF), g=torch.zeros(E, I, H, dtype=BF), u=torch.zeros(E, I, H, dtype=BF),
             d=torch.zeros(E, H, I, dtype=BF), limit=None, first=0)
    a.update(kw)
    return F.forward_few_tokens(a["x"], a["top"], a["w"], a["sg"], a["su"], a["sd"], a["g"], a["u"], a["d"], a["limit"], first_expert=a["first"])


def test_few_tokens_arguments():
    with pytest.raises(ValueError, match="CUDA tensor"):
        few()
    f8, u8 = torch.zeros(2, 128, 256, dtype=torch.float8_e4m3fn), torch.zeros(2, 2, 32, 16, dtype=torch.uint8)
    for kw, error, why in (
            (dict(T=512), ValueError, "at most 511"), (dict(H=128), ValueError, "hidden_size"), (dict(I=64), ValueError, "intermediate_size"),
            (dict(x=torch.zeros(256, dtype=BF)), ValueError, "x must have shape"), (dict(x=torch.zeros(4, 256)), TypeError, "x must have dtype"),
            (dict(top=torch.zeros(4, dtype=I64)), ValueError, "top_experts"), (dict(top=torch.zeros(4, 256, dtype=I64)), ValueError, "topk"),
            (dict(limit=-1.0), ValueError, "swiglu_limit"), (dict(limit=float("nan")), ValueError, "swiglu_limit"), (dict(first=-1), ValueError, "first_expert"),
            (dict(first=0.0), ValueError, "first_expert"), (dict(g=torch.zeros(128, 256, dtype=BF)), ValueError, "w_routed_gate"),
            (dict(g=(f8, u8)), TypeError, "same precision"), (dict(g=(f8, u8, f8), u=(f8, u8), d=(f8, u8)), ValueError, "pairs")):
        with pytest.raises(error, match=why):
            few(**kw)


def test_packed_arguments():
    from mok import functional as F, ops
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.pack_rows(torch.zeros(2, 128, dtype=BF))
    with pytest.raises(ValueError, match="divisible by 16"):
        ops.pack_rows(torch.zeros(2, 120, dtype=BF))
    with pytest.raises(ValueError, match="shape"):
        ops.pack_rows(torch.zeros(128, dtype=BF))
    with pytest.raises(TypeError, match="dtype"):
        ops.pack_rows(torch.zeros(2, 128))
    q, s = torch.zeros(2, 256, dtype=I8), torch.zeros(2, 2)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.unpack_rows(q, s)
    with pytest.raises(TypeError, match="dtype"):
        ops.unpack_rows(q.to(torch.uint8), s)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.swiglu_bwd_packed(q, s, q, s, torch.zeros(2, 256, dtype=BF))
    with pytest.raises(TypeError, match="MoKSchedule"):
        F.pack_context(None, None)
    t = torch.zeros(2, 128, dtype=BF)
    sched = F.MoKSchedule(peer_rank=t, peer_token_idx=t, num_tokens=t, tokens_per_expert=t)
    with pytest.raises(TypeError, match="MoKForwardContext"):
        F.pack_context(sched, None)
    ctx = F.MoKForwardContext(x_routed=(t, t), gate_shared=t, gate_routed=(t, t), up_shared=t, up_routed=(t, t), hidden_shared=t, hidden_routed=(t, t))
    with pytest.raises(TypeError, match="in 8 bits already"):
        F.pack_context(sched, ctx)


def test_the_library_checks_sizes_and_addresses():
    """Addresses here are numbers that nothing reads: every call returns before it launches."""
    from mok import _C
    lib, a = _C.lib, ctypes.c_void_p(4096)
    def refused(rc, why):
        assert rc == -1 and why in _C._last_error(), (rc, _C._last_error())
    route = lambda E=16, K=2, ld=16, score=0, bias=None, counts=None, sums=None, scratch=None, scale=1.0, T=4, l=a: lib.mokb_route(
        l, 0, ld, T, E, K, score, bias, 1, scale, a, a, counts, sums, scratch, None)
    refused(route(E=1025, ld=1025), b"num_experts")
    refused(route(K=17), b"topk")
    refused(route(K=0), b"topk")
    refused(route(ld=15), b"stride")
    refused(route(score=2), b"score")
    refused(route(bias=a), b"sigmoid")
    refused(route(counts=a), b"together")
    refused(route(counts=a, sums=a), b"scratch")
    refused(route(scale=float("nan")), b"scale")
    refused(route(l=None), b"null")
    assert route(T=0) == 0
    refused(lib.mokb_route_bwd(a, 0, 16, 4, 16, 2, 0, 1, 1.0, None, a, None, a, None), b"null")
    assert lib.mokb_route_scratch_bytes(4, 1025) == 0 and lib.mokb_route_scratch_bytes(100000, 256) > 256 * 8

    def args(**kw):
        f = _C.FewTokensArgs(num_tokens=4, hidden=256, intermediate=128, num_local_experts=2, topk=2)
        for n in ("x", "top_experts", "router_weights", "w_routed_gate", "w_routed_up", "w_routed_down", "y", "workspace", "status"):
            setattr(f, n, 4096)
        for n, v in kw.items():
            setattr(f, n, v)
        return ctypes.byref(f)
    few_fwd = lambda **kw: lib.mokb_few_tokens_fwd(args(**kw), None)
    refused(lib.mokb_few_tokens_fwd(None, None), b"null args")
    refused(few_fwd(num_tokens=512), b"num_tokens")
    refused(few_fwd(num_tokens=-1), b"num_tokens")
    refused(few_fwd(hidden=384), b"hidden")
    refused(few_fwd(intermediate=64), b"intermediate")
    refused(few_fwd(topk=0), b"topk")
    refused(few_fwd(num_local_experts=0), b"num_local_experts")
    refused(few_fwd(first_expert=-1), b"first_expert")
    refused(few_fwd(x=4100), b"16-byte")
    refused(few_fwd(workspace=4112), b"256-byte")
    refused(few_fwd(y=None), b"null pointer")
    refused(few_fwd(w_routed_up=None), b"null weight")
    refused(few_fwd(w_shared_up=4096), b"together")
    refused(few_fwd(mxfp8=1), b"null scales")
    refused(few_fwd(num_local_experts=4097), b"num_local_experts")
    assert few_fwd(num_tokens=0) == 0
    assert lib.mokb_few_tokens_workspace_bytes(512, 256, 128, 2, 0) == 0 and lib.mokb_few_tokens_workspace_bytes(1, 256, 128, 2, 0) > 0

    refused(lib.mokb_pack_rows(a, a, a, None, 4, 100, None), b"multiple of 16")
    refused(lib.mokb_pack_rows(ctypes.c_void_p(4112), a, a, None, 4, 128, None), b"aligned")
    refused(lib.mokb_pack_rows(a, None, a, None, 4, 128, None), b"null")
    refused(lib.mokb_unpack_rows(a, a, ctypes.c_void_p(4112), None, 4, 128, None), b"aligned")
    refused(lib.mokb_unpack_rows(a, a, a, None, -1, 128, None), b"multiple of 16")
    refused(lib.mokb_swiglu_bwd_packed(a, a, a, a, a, a, a, None, None, None, None, 4, 128, 0, 0.0, None), b"null")
    refused(lib.mokb_swiglu_bwd_packed(a, a, a, a, a, a, a, ctypes.c_void_p(4112), None, None, None, 4, 128, 0, 0.0, None), b"aligned")
    refused(lib.mokb_swiglu_bwd_packed(a, a, a, a, a, a, a, a, None, None, None, 4, 131088, 0, 0.0, None), b"131072")
    assert lib.mokb_pack_rows(None, None, None, None, 0, 128, None) == 0
    b = _C.BwdArgs()
    refused(lib.mokb_dispatch_mlp_swiglu_combine_bwd_bf16_packed(ctypes.byref(b), None, None), b"null packed context")


def test_fake_kernels_give_the_shapes():
    """Under FakeTensorMode, as torch.compile traces them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from mok import functional as F, ops
    with FakeTensorMode():
        t = lambda *s, dtype=BF: torch.empty(s, dtype=dtype)
        r = F.route(F.MoKRouterConfig(topk=3), t(5, 8, dtype=F32), balance=True)
        assert r.top_experts.shape == (5, 3) and r.top_experts.dtype == I64 and r.score_sums.shape == (8,) and r.tokens_per_expert.dtype == torch.int32
        assert F.route(F.MoKRouterConfig(topk=3), t(5, 8)).score_sums is None
        assert F.route_backward(F.MoKRouterConfig(topk=3), t(5, 8), r, t(5, 3, dtype=F32)).dtype == BF
        y = F.forward_few_tokens(t(4, 256), t(4, 2, dtype=I64), t(4, 2, dtype=F32), None, None, None, t(2, 128, 256), t(2, 128, 256), t(2, 256, 128))
        assert y.shape == (4, 256)
        q, s = ops.pack_rows(t(3, 272))
        assert q.shape == (3, 272) and q.dtype == I8 and s.shape == (3, 3)
        assert ops.unpack_rows(q, s).dtype == BF
        outs = ops.swiglu_bwd_packed(q, s, q, s, t(3, 272))
        assert [tuple(o.shape) for o in outs] == [(3, 272)] * 3 + [(3,)]
