"""The operators of `mok.ops` around the layer: the router and its gradient, the whole layer for a few tokens, and activations
kept in 8 bits between the forward and the backward pass.  The reference has none of them (its layer starts from given routes,
takes 512 tokens or more and saves bf16 or MXFP8); the manner is that of its other operators: arguments are checked before any
device work (ValueError / TypeError), outputs are allocated, nothing synchronises the host.  `mok.ops` re-exports them."""
import torch

from . import _C
from . import ops as _ops
from .ops_mxfp8 import F8, _sc_shape

MAX_FEW_TOKENS = 511
MAX_FEW_EXPERTS = 4096
MAX_ROUTE_EXPERTS = 1024
MAX_ROUTE_TOPK = 32
PACK_BLOCK = _C.PACK_BLOCK

BF16, F32, I64 = torch.bfloat16, torch.float32, torch.int64
FLT_MAX = torch.finfo(torch.float32).max


def _check_cuda(name: str, t: torch.Tensor, dtype, shape=None, device=None, contiguous=True) -> None:
    """A tensor of the current CUDA device (kernels go to that device's current stream), of `dtype` and `shape`, without gaps."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise TypeError(f"{name} must have dtype {dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if device is None and t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} must be on the current CUDA device")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _plain(t, dtype, shape, device) -> bool:
    """What `_check_cuda` accepts, asked in one go: the detailed checks only have to name what is wrong."""
    return isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device and t.is_contiguous()


def _here(t, dtype) -> bool:
    """A CUDA tensor of the current device, of `dtype`: the short way past `_check_cuda` (a host microsecond counts in a small call)."""
    return isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda and t.get_device() == torch.cuda.current_device()


def _check_limit(swiglu_limit) -> None:
    if swiglu_limit is not None and (type(swiglu_limit) not in (int, float) or not swiglu_limit >= 0):
        raise ValueError("swiglu_limit must be None or a non-negative number")


# ---------------------------------------------------------------------------------------------------------------- router
def check_route_knobs(topk, score, renormalize, scale) -> None:
    if type(topk) is not int or not 0 < topk <= MAX_ROUTE_TOPK:
        raise ValueError(f"topk must be an integer in [1, {MAX_ROUTE_TOPK}]")
    if score not in ("softmax", "sigmoid"):
        raise ValueError("score must be 'softmax' or 'sigmoid'")
    if type(renormalize) is not bool:
        raise TypeError("renormalize must be a boolean")
    if type(scale) not in (int, float) or not abs(scale) <= FLT_MAX:
        raise ValueError("scale must be a finite number of fp32's range")


def _check_logits(logits, topk, score, renormalize, scale) -> tuple[int, int]:
    check_route_knobs(topk, score, renormalize, scale)
    if not isinstance(logits, torch.Tensor) or logits.ndim != 2:
        raise ValueError("logits must have shape (num_tokens, num_experts)")
    T, E = logits.shape
    if not topk <= E <= MAX_ROUTE_EXPERTS:
        raise ValueError(f"num_experts must be in [topk, {MAX_ROUTE_EXPERTS}]")
    if not (_here(logits, F32) or _here(logits, BF16)):
        _check_cuda("logits", logits, (F32, BF16), contiguous=False)
    if (E > 1 and logits.stride(1) != 1) or (T > 1 and logits.stride(0) < E):
        raise ValueError("the logits of a token must be contiguous and tokens must not overlap")
    return T, E


@_ops._op(
    "mok::route", mutates_args=(),
    schema="(Tensor logits, Tensor? bias, int topk, str score, bool renormalize, float scale, bool balance) -> (Tensor, Tensor, Tensor?, Tensor?)",
)
def route(logits, bias, topk, score, renormalize, scale, balance):
    """[num_tokens, num_experts] logits (fp32 or bf16; rows may be apart) -> top_experts [T, topk] int64, router_weights [T, topk]
    fp32 and, with `balance`, tokens_per_expert [E] int32 and score_sums [E] fp32 (else None, None).

    score "softmax": the largest logits are picked; "sigmoid": the largest 1 / (1 + exp(-logit)) + bias (`bias` [E] fp32, finite,
    only picks, has no gradient; where the sum is NaN or -inf the expert comes last).  Weights are the scores of the picks times `scale`, with `renormalize` divided by their sum.
    Ties go to the lowest index.  Logits that are -inf or NaN close an expert for the token: picked only when nothing else is left,
    with weight 0; not counted in the load figures."""
    T, E = _check_logits(logits, topk, score, renormalize, scale)
    if bias is not None:
        if score != "sigmoid":
            raise ValueError("a bias goes with score 'sigmoid'")
        if not _plain(bias, F32, (E,), logits.device):
            _check_cuda("bias", bias, F32, (E,), logits.device)
    if type(balance) is not bool:
        raise TypeError("balance must be a boolean")
    return _C.route(logits, bias, topk, score == "sigmoid", renormalize, float(scale), balance)


@_ops._op("mok::route_bwd", mutates_args=())
def route_bwd(
    logits: torch.Tensor,
    top_experts: torch.Tensor,
    d_router_weights: torch.Tensor,
    d_score_sums: torch.Tensor | None,
    score: str,
    renormalize: bool,
    scale: float,
) -> torch.Tensor:
    """The gradient of the logits, in their type, from that of the router weights [T, topk] fp32 and (optional) of score_sums [E]
    fp32; top_experts as `route` returned them.  The picks are constants."""
    topk = top_experts.shape[1] if isinstance(top_experts, torch.Tensor) and top_experts.ndim == 2 else 0
    if topk == 0:
        raise ValueError("top_experts must have shape (num_tokens, topk)")
    T, E = _check_logits(logits, topk, score, renormalize, scale)
    dev = logits.device
    if not (_plain(top_experts, I64, (T, topk), dev) and _plain(d_router_weights, F32, (T, topk), dev)):
        _check_cuda("top_experts", top_experts, I64, (T, topk), dev)
        _check_cuda("d_router_weights", d_router_weights, F32, (T, topk), dev)
    if d_score_sums is not None and not _plain(d_score_sums, F32, (E,), dev):
        _check_cuda("d_score_sums", d_score_sums, F32, (E,), dev)
    return _C.route_bwd(logits, top_experts, d_router_weights, d_score_sums, score == "sigmoid", renormalize, float(scale))


# ---------------------------------------------------------------------------------------------------------------- few tokens
@_ops._op("mok::few_tokens_fwd", mutates_args=())
def few_tokens_fwd(
    x: torch.Tensor,
    top_experts: torch.Tensor,
    router_weights: torch.Tensor,
    w_shared_gate: torch.Tensor | None,
    w_shared_up: torch.Tensor | None,
    w_shared_down: torch.Tensor | None,
    w_routed_gate: torch.Tensor,
    w_routed_gate_sc: torch.Tensor | None,
    w_routed_up: torch.Tensor,
    w_routed_up_sc: torch.Tensor | None,
    w_routed_down: torch.Tensor,
    w_routed_down_sc: torch.Tensor | None,
    first_expert: int,
    swiglu_limit: float | None,
) -> torch.Tensor:
    """The whole layer for 0 to 511 tokens on this rank's experts [first_expert, first_expert + num_local_experts):
    y = shared(x) + sum_k router_weights[:, k] * expert_{top_experts[:, k]}(x).  Routes to other experts and routes of weight 0
    contribute nothing; the three shared weights may be None together.  With scales the routed weights are E4M3, as
    `mxfp8_quantize` returns them, and x and hidden are quantised likewise."""
    if not isinstance(x, torch.Tensor) or x.ndim != 2:
        raise ValueError("x must have shape (num_tokens, hidden_size)")
    T, H = x.shape
    if T > MAX_FEW_TOKENS:
        raise ValueError(f"num_tokens must be at most {MAX_FEW_TOKENS}: the layer with a schedule takes more")
    if H <= 0 or H % 256 != 0:
        raise ValueError("hidden_size must be positive and divisible by 256")
    if not isinstance(w_routed_gate, torch.Tensor) or w_routed_gate.ndim != 3 or w_routed_gate.shape[0] <= 0:
        raise ValueError("w_routed_gate must have shape (num_local_experts, intermediate_size, hidden_size)")
    E, I, _ = w_routed_gate.shape
    if E > MAX_FEW_EXPERTS:
        raise ValueError(f"num_local_experts must be at most {MAX_FEW_EXPERTS}")
    if I <= 0 or I % 128 != 0:
        raise ValueError("intermediate_size must be positive and divisible by 128")
    if not isinstance(top_experts, torch.Tensor) or top_experts.ndim != 2 or not 0 < top_experts.shape[1] <= 255:
        raise ValueError("top_experts must have shape (num_tokens, topk) with topk in [1, 255]")
    K = top_experts.shape[1]
    if type(first_expert) is not int or not 0 <= first_expert < 2 ** 31:
        raise ValueError("first_expert must be a non-negative integer")
    if swiglu_limit is not None:
        _check_limit(swiglu_limit)
    if not (_here(x, BF16) and x.is_contiguous()):
        _check_cuda("x", x, BF16)
    dev = x.device
    mx = w_routed_gate_sc is not None
    if (w_routed_up_sc is not None) != mx or (w_routed_down_sc is not None) != mx:
        raise ValueError("the scales of the routed weights go together")
    shared = w_shared_gate is not None
    if (w_shared_up is not None) != shared or (w_shared_down is not None) != shared:
        raise ValueError("the shared expert's weights go together")
    wt = F8 if mx else BF16
    routed, routed_down = (E, I, H), (E, H, I)
    if not (_plain(top_experts, I64, (T, K), dev) and _plain(router_weights, F32, (T, K), dev) and _plain(w_routed_gate, wt, routed, dev)
            and _plain(w_routed_up, wt, routed, dev) and _plain(w_routed_down, wt, routed_down, dev)):
        for name, t, dtype, shape in (("top_experts", top_experts, I64, (T, K)), ("router_weights", router_weights, F32, (T, K)),
                                      ("w_routed_gate", w_routed_gate, wt, routed), ("w_routed_up", w_routed_up, wt, routed),
                                      ("w_routed_down", w_routed_down, wt, routed_down)):
            _check_cuda(name, t, dtype, shape, dev)
    if mx:
        for name, t, rows, cols in (("w_routed_gate_sc", w_routed_gate_sc, I, H), ("w_routed_up_sc", w_routed_up_sc, I, H),
                                    ("w_routed_down_sc", w_routed_down_sc, H, I)):
            if not _plain(t, torch.uint8, _sc_shape(E * rows, cols), dev):
                _check_cuda(name, t, torch.uint8, _sc_shape(E * rows, cols), dev)
    if shared and not (_plain(w_shared_gate, BF16, (I, H), dev) and _plain(w_shared_up, BF16, (I, H), dev) and _plain(w_shared_down, BF16, (H, I), dev)):
        for name, t, shape in (("w_shared_gate", w_shared_gate, (I, H)), ("w_shared_up", w_shared_up, (I, H)), ("w_shared_down", w_shared_down, (H, I))):
            _check_cuda(name, t, BF16, shape, dev)
    if T == 0:
        return torch.empty_like(x)
    return _C.few_tokens_fwd(x, top_experts, router_weights, w_shared_gate, w_shared_up, w_shared_down, w_routed_gate, w_routed_up,
                             w_routed_down, (w_routed_gate_sc, w_routed_up_sc, w_routed_down_sc) if mx else None, first_expert, swiglu_limit)


# ---------------------------------------------------------------------------------------------------------------- 8-bit activations
def _check_rows(name: str, rows: int, cols: int) -> None:
    if cols <= 0 or cols % 16 != 0:
        raise ValueError(f"{name}'s number of columns must be positive and divisible by 16")


def _check_num_rows(num_rows, device) -> None:
    if num_rows is not None:
        _check_cuda("num_rows", num_rows, torch.int32, (1,), device)


def _check_packed(name: str, q, scales, device=None) -> tuple[int, int]:
    if not isinstance(q, torch.Tensor) or q.ndim != 2:
        raise ValueError(f"{name} must have shape (rows, columns)")
    rows, cols = q.shape
    _check_rows(name, rows, cols)
    shape = (rows, -(-cols // PACK_BLOCK))
    if not (_here(q, torch.int8) and q.is_contiguous() and (device is None or q.device == device) and _plain(scales, F32, shape, q.device)):
        _check_cuda(name, q, torch.int8, None, device)
        _check_cuda(f"{name}'s scales", scales, F32, shape, q.device)
    return rows, cols


@_ops._op("mok::pack_rows", mutates_args=())
def pack_rows_op(x: torch.Tensor, num_rows: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 [rows, columns] -> q int8 and scales [rows, ceil(columns / 128)] fp32: x ~ q * scale, one scale per 128 values of a row,
    off by half a step of max|x| / 127 at most.  With `num_rows` (int32 [1] on the device, e.g. a schedule's num_tokens) only the
    first num_rows rows are packed and the others are left unwritten."""
    if not isinstance(x, torch.Tensor) or x.ndim != 2:
        raise ValueError("x must have shape (rows, columns)")
    _check_rows("x", *x.shape)
    if not (_here(x, BF16) and x.is_contiguous()):
        _check_cuda("x", x, BF16)
    if num_rows is not None:
        _check_num_rows(num_rows, x.device)
    return _C.pack_rows(x, num_rows)


@_ops._op("mok::unpack_rows", mutates_args=())
def unpack_rows_op(q: torch.Tensor, scales: torch.Tensor, num_rows: torch.Tensor | None = None) -> torch.Tensor:
    """What `pack_rows` kept, as bf16."""
    _check_packed("q", q, scales)
    if num_rows is not None:
        _check_num_rows(num_rows, q.device)
    return _C.unpack_rows(q, scales, num_rows)


@_ops._op("mok::swiglu_bwd_packed", mutates_args=())
def swiglu_bwd_packed_op(
    gate_q: torch.Tensor,
    gate_scales: torch.Tensor,
    up_q: torch.Tensor,
    up_scales: torch.Tensor,
    d_hidden: torch.Tensor,
    swiglu_limit: float | None = None,
    row_scale: torch.Tensor | None = None,
    num_rows: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The backward pass of hidden = silu(gate) * up from packed gate and up: d_gate, d_up, hidden (bf16) and per row
    sum(d_hidden * hidden) / row_scale (0 where row_scale is not positive; without row_scale, the sum). At most 131072 columns."""
    shape = _check_packed("gate_q", gate_q, gate_scales)
    if _check_packed("up_q", up_q, up_scales, gate_q.device) != shape:
        raise ValueError("gate and up must have the same shape")
    _check_cuda("d_hidden", d_hidden, BF16, shape, gate_q.device)
    _check_limit(swiglu_limit)
    if row_scale is not None:
        _check_cuda("row_scale", row_scale, F32, shape[:1], gate_q.device)
    _check_num_rows(num_rows, gate_q.device)
    return _C.swiglu_bwd_packed(gate_q, gate_scales, up_q, up_scales, d_hidden, swiglu_limit, row_scale, num_rows)


# The three above are called as they are, also many times a step, so the public names take the short way that `call` knows.
def pack_rows(x, num_rows=None):
    return _ops.call(pack_rows_op, x, num_rows)


def unpack_rows(q, scales, num_rows=None):
    return _ops.call(unpack_rows_op, q, scales, num_rows)


def swiglu_bwd_packed(gate_q, gate_scales, up_q, up_scales, d_hidden, swiglu_limit=None, row_scale=None, num_rows=None):
    return _ops.call(swiglu_bwd_packed_op, gate_q, gate_scales, up_q, up_scales, d_hidden, swiglu_limit, row_scale, num_rows)


for _f, _o in ((pack_rows, pack_rows_op), (unpack_rows, unpack_rows_op), (swiglu_bwd_packed, swiglu_bwd_packed_op)):
    _f.__doc__ = _ops._EAGER[_o][0].__doc__


@_ops._op(
    "mok::dispatch_mlp_swiglu_combine_bwd_bf16_packed", mutates_args=("d_x_routed_buffer", "d_router_weight_buffer"),
)
def dispatch_mlp_swiglu_combine_bwd_bf16_packed(
    d_y_buffer: torch.Tensor,
    d_y_buffer_ptrs: list[int],
    d_x_routed_buffer: torch.Tensor,
    d_x_routed_buffer_ptrs: list[int],
    router_weight_buffer: torch.Tensor,
    router_weight_buffer_ptrs: list[int],
    d_router_weight_buffer: torch.Tensor,
    d_router_weight_buffer_ptrs: list[int],
    w_shared_gate: torch.Tensor,
    w_routed_gate: torch.Tensor,
    w_shared_up: torch.Tensor,
    w_routed_up: torch.Tensor,
    w_shared_down: torch.Tensor,
    w_routed_down: torch.Tensor,
    x_routed_q: torch.Tensor,
    x_routed_scales: torch.Tensor,
    gate_routed_q: torch.Tensor,
    gate_routed_scales: torch.Tensor,
    up_routed_q: torch.Tensor,
    up_routed_scales: torch.Tensor,
    gate_shared_q: torch.Tensor,
    gate_shared_scales: torch.Tensor,
    up_shared_q: torch.Tensor,
    up_shared_scales: torch.Tensor,
    x: torch.Tensor,
    x_ptrs: list[int],
    schedule_peer_rank: torch.Tensor,
    schedule_peer_token_idx: torch.Tensor,
    num_tokens: torch.Tensor,
    tokens_per_expert: torch.Tensor,
    topk: int,
    swiglu_limit: float | None,
    num_comm_sms: int,
    macrobatch_size: int,
    minibatch_size: int,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
           torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
           torch.Tensor]:
    """`dispatch_mlp_swiglu_combine_bwd_bf16` from a packed context (x_routed [MB, H], gate and up of the routed rows [MB, I] and of
    the shared expert [T, I]); same outputs.  The context is left as it is."""
    T, H = _ops._check_activation("x", x)
    I, E_l = _ops._check_weights(w_shared_gate, w_routed_gate, H)
    _ops._check_knobs(topk, swiglu_limit, num_comm_sms, macrobatch_size, minibatch_size)
    ep_size = _ops._check_ptrs("x_ptrs", x_ptrs)
    for name, ptrs in (("d_y_buffer_ptrs", d_y_buffer_ptrs), ("d_x_routed_buffer_ptrs", d_x_routed_buffer_ptrs),
                       ("router_weight_buffer_ptrs", router_weight_buffer_ptrs),
                       ("d_router_weight_buffer_ptrs", d_router_weight_buffer_ptrs)):
        _ops._check_ptrs(name, ptrs, ep_size)
    _ops._check_schedule(schedule_peer_rank, schedule_peer_token_idx, num_tokens, tokens_per_expert, E_l)
    MB = macrobatch_size
    _ops._check_shapes_devices(x.device, [
        ("d_y_buffer", d_y_buffer, (T, H)), ("d_x_routed_buffer", d_x_routed_buffer, (T * topk, H)),
        ("router_weight_buffer", router_weight_buffer, (T, topk)),
        ("d_router_weight_buffer", d_router_weight_buffer, (T, topk)),
        ("w_shared_gate", w_shared_gate, (I, H)), ("w_routed_gate", w_routed_gate, (E_l, I, H)),
        ("w_shared_up", w_shared_up, (I, H)), ("w_routed_up", w_routed_up, (E_l, I, H)),
        ("w_shared_down", w_shared_down, (H, I)), ("w_routed_down", w_routed_down, (E_l, H, I)),
        ("schedule_peer_rank", schedule_peer_rank, None), ("schedule_peer_token_idx", schedule_peer_token_idx, None),
        ("num_tokens", num_tokens, None), ("tokens_per_expert", tokens_per_expert, None),
    ])
    packed = (x_routed_q, x_routed_scales, gate_routed_q, gate_routed_scales, up_routed_q, up_routed_scales,
              gate_shared_q, gate_shared_scales, up_shared_q, up_shared_scales)
    for i, (name, shape) in enumerate((("x_routed_q", (MB, H)), ("gate_routed_q", (MB, I)), ("up_routed_q", (MB, I)),
                                       ("gate_shared_q", (T, I)), ("up_shared_q", (T, I)))):
        if _check_packed(name, packed[2 * i], packed[2 * i + 1], x.device) != shape:
            raise ValueError(f"{name} must have shape {shape}")
    return _C.dispatch_mlp_swiglu_combine_bwd_bf16_packed(
        d_y_buffer, d_y_buffer_ptrs, d_x_routed_buffer, d_x_routed_buffer_ptrs, router_weight_buffer,
        router_weight_buffer_ptrs, d_router_weight_buffer, d_router_weight_buffer_ptrs, w_shared_gate, w_routed_gate,
        w_shared_up, w_routed_up, w_shared_down, w_routed_down, packed, x, x_ptrs, schedule_peer_rank,
        schedule_peer_token_idx, num_tokens, tokens_per_expert, topk, swiglu_limit, num_comm_sms, macrobatch_size,
        minibatch_size)


# ---------------------------------------------------------------------------------------------------------------- fake kernels
def _register_fakes() -> None:
    fake = torch.library.register_fake

    @fake("mok::route")
    def _(logits, bias, topk, score, renormalize, scale, balance):
        T, E = logits.shape
        return (logits.new_empty((T, topk), dtype=I64), logits.new_empty((T, topk), dtype=F32),
                logits.new_empty((E,), dtype=torch.int32) if balance else None, logits.new_empty((E,), dtype=F32) if balance else None)

    @fake("mok::route_bwd")
    def _(logits, top_experts, d_router_weights, d_score_sums, score, renormalize, scale):
        return logits.new_empty(tuple(logits.shape))

    @fake("mok::few_tokens_fwd")
    def _(x, top_experts, router_weights, w_shared_gate, w_shared_up, w_shared_down, w_routed_gate, w_routed_gate_sc, w_routed_up,
          w_routed_up_sc, w_routed_down, w_routed_down_sc, first_expert, swiglu_limit):
        return torch.empty_like(x)

    def packed(x):
        rows, cols = x.shape
        return x.new_empty((rows, cols), dtype=torch.int8), x.new_empty((rows, -(-cols // PACK_BLOCK)), dtype=F32)

    @fake("mok::pack_rows")
    def _(x, num_rows=None):
        return packed(x)

    @fake("mok::unpack_rows")
    def _(q, scales, num_rows=None):
        return q.new_empty(tuple(q.shape), dtype=BF16)

    @fake("mok::swiglu_bwd_packed")
    def _(gate_q, gate_scales, up_q, up_scales, d_hidden, swiglu_limit=None, row_scale=None, num_rows=None):
        return (*(torch.empty_like(d_hidden) for _ in range(3)), d_hidden.new_empty((d_hidden.shape[0],), dtype=F32))

    @fake("mok::dispatch_mlp_swiglu_combine_bwd_bf16_packed")
    def _(d_y_buffer, d_y_buffer_ptrs, d_x_routed_buffer, d_x_routed_buffer_ptrs, router_weight_buffer,
          router_weight_buffer_ptrs, d_router_weight_buffer, d_router_weight_buffer_ptrs, w_shared_gate, w_routed_gate,
          w_shared_up, w_routed_up, w_shared_down, w_routed_down, x_routed_q, x_routed_scales, gate_routed_q,
          gate_routed_scales, up_routed_q, up_routed_scales, gate_shared_q, gate_shared_scales, up_shared_q,
          up_shared_scales, x, x_ptrs, schedule_peer_rank, schedule_peer_token_idx, num_tokens, tokens_per_expert, topk,
          swiglu_limit, num_comm_sms, macrobatch_size, minibatch_size):
        T, H = x.shape
        E_l, I = w_routed_gate.shape[:2]
        MB = macrobatch_size

        def bf(*shape):
            return x.new_empty(shape, dtype=BF16)
        return (bf(T, H), bf(MB, H), bf(T, I), bf(MB, I), bf(T, I), bf(MB, I), bf(T, I), bf(MB, I), bf(MB, H), bf(I, H),
                bf(E_l, I, H), bf(I, H), bf(E_l, I, H), bf(H, I), bf(E_l, H, I))


_register_fakes()
