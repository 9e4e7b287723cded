"""torch.library.opcheck on the operators around the layer: schemas, fake kernels and tracing agree with what they do."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CHECKS = ("test_schema", "test_faketensor")


def test_opcheck():
    from mok import ops  # noqa: F401
    from tests.test_gpu_few_tokens import make
    m = torch.ops.mok
    logits = torch.randn(20, 24, device="cuda")
    for args in ((logits, None, 4, "softmax", True, 1.0, True), (logits.bfloat16(), torch.zeros(24, device="cuda"), 4, "sigmoid", False, 2.0, False)):
        torch.library.opcheck(m.route.default, args, test_utils=CHECKS)
    top = m.route(logits, None, 4, "softmax", True, 1.0, False)[0]
    torch.library.opcheck(m.route_bwd.default, (logits, top, torch.randn(20, 4, device="cuda"), torch.zeros(24, device="cuda"), "softmax", True, 1.0),
                          test_utils=CHECKS)
    x, t, w, sh, routed = make(5, 256, 128, 4, 2)
    torch.library.opcheck(m.few_tokens_fwd.default, (x, t, w, *sh, routed[0], None, routed[1], None, routed[2], None, 0, 2.0), test_utils=CHECKS)
    x, t, w, sh, routed = make(5, 256, 128, 4, 2, mx=True)
    torch.library.opcheck(m.few_tokens_fwd.default, (x, t, w, None, None, None, *routed[0], *routed[1], *routed[2], 0, None),
                           test_utils="test_faketensor")      # (the schema check does not know E4M3 tensors)
    v = torch.randn(6, 160, device="cuda").bfloat16()
    torch.library.opcheck(m.pack_rows.default, (v, None), test_utils=CHECKS)
    q, s = m.pack_rows(v)
    torch.library.opcheck(m.unpack_rows.default, (q, s, None), test_utils=CHECKS)
    torch.library.opcheck(m.swiglu_bwd_packed.default, (q, s, q, s, v, None, torch.ones(6, device="cuda"), None), test_utils=CHECKS)


def test_refusals_of_tensors_on_the_gpu():
    """What only a CUDA tensor gets as far as: other types, shapes, places and gaps, before any launch."""
    from mok import _C, functional as F, ops
    from tests.test_gpu_few_tokens import make
    before = _C.launch_count()
    logits = torch.randn(8, 16, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        ops.route(logits.t().contiguous().t(), None, 2, "softmax", True, 1.0, False)
    with pytest.raises(ValueError, match="overlap"):
        ops.route(logits[:1].expand(8, 16), None, 2, "softmax", True, 1.0, False)
    with pytest.raises(ValueError, match="bias must be a CUDA tensor"):
        ops._EAGER[ops.route][0](logits, torch.zeros(16), 2, "sigmoid", True, 1.0, False)
    with pytest.raises(ValueError, match="sigmoid"):
        ops._EAGER[ops.route][0](logits, torch.zeros(16, device="cuda"), 2, "softmax", True, 1.0, False)
    with pytest.raises(TypeError, match="top_experts"):
        F.route_backward(F.MoKRouterConfig(topk=2), logits, F.MoKRouting(torch.zeros(8, 2, dtype=torch.int32, device="cuda"), None, None, None),
                         torch.zeros(8, 2, device="cuda"))
    with pytest.raises(ValueError, match="d_router_weights"):
        F.route_backward(F.MoKRouterConfig(topk=2), logits, F.MoKRouting(torch.zeros(8, 2, dtype=torch.int64, device="cuda"), None, None, None),
                         torch.zeros(8, 3, device="cuda"))
    x, t, w, sh, r = make(4, 256, 128, 4, 2)
    few = F.forward_few_tokens
    with pytest.raises(ValueError, match="x must be contiguous"):
        few(x.t().contiguous().t(), t, w, *sh, *r)
    with pytest.raises(TypeError, match="top_experts"):
        few(x, t.int(), w, *sh, *r)
    with pytest.raises(ValueError, match="router_weights"):
        few(x, t, w[:, :1].contiguous(), *sh, *r)
    with pytest.raises(ValueError, match="w_routed_down"):
        few(x, t, w, *sh, r[0], r[1], r[1])
    with pytest.raises(ValueError, match="go together"):
        few(x, t, w, sh[0], None, sh[2], *r)
    with pytest.raises(TypeError, match="w_shared_up"):
        few(x, t, w, sh[0], sh[1].float(), sh[2], *r)
    v = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        ops.pack_rows(v[:, :128])
    with pytest.raises(_C.MokError, match="32-byte"):
        ops.pack_rows(torch.zeros(4 * 256 + 8, dtype=torch.bfloat16, device="cuda")[8:].view(4, 256))
    with pytest.raises(TypeError, match="num_rows"):
        ops.pack_rows(v, torch.zeros(1, dtype=torch.int64, device="cuda"))
    q, s = torch.zeros(4, 256, dtype=torch.int8, device="cuda"), torch.zeros(4, 2, device="cuda")
    with pytest.raises(ValueError, match="scales"):
        ops.unpack_rows(q, s[:, :1].contiguous())
    with pytest.raises(ValueError, match="same shape"):
        ops.swiglu_bwd_packed(q, s, q[:3], s[:3], v)
    with pytest.raises(ValueError, match="d_hidden"):
        ops.swiglu_bwd_packed(q, s, q, s, v[:3])
    assert _C.launch_count() == before
