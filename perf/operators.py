"""Operators around the MoE layer: the router with its gradient, the layer for a few tokens, activations kept in 8 bits.

A case is a dict of plain values with an "op":
  "route"    the router: top-k experts and weights of every token, the load figures, and (backward) the gradient of the logits
  "few"      the whole layer, shared expert included, for the few tokens of a decoding step, bf16 or MXFP8 routed weights
  "restore"  a saved activation: packed in the forward pass, unpacked in the backward pass
  "swiglu8"  gate and up packed in the forward pass; the backward pass of SwiGLU from the packed values, hidden included

`own` False computes the plain forms below, True calls `mok.functional` and `mok.ops`.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 128             # values of a row that share one scale of the 8-bit activations


# ---------------------------------------------------------------------------------------------------- cases
def _route(name, tokens, experts, topk, score, bias=False, renorm=True, scale=1.0, dtype="fp32", masked=0.0, backward=True):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "topk": topk, "score": score, "bias": bias,
            "renorm": renorm, "scale": scale, "dtype": dtype, "masked": masked, "backward": backward}


def _few(name, precision, tokens, hidden, inter, experts, topk, ranks=1, shared=True, limit=0.0, padded=0.0):
    """`ranks`: the router chooses among ranks * experts, of which this one holds `experts`; `padded`: share of tokens without weight."""
    return {"name": name, "op": "few", "precision": precision, "tokens": tokens, "hidden": hidden, "inter": inter, "experts": experts,
            "topk": topk, "ranks": ranks, "shared": shared, "limit": limit, "padded": padded}


def _packed(name, op, rows, cols, limit=0.0):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "limit": limit}


def listed():
    return [
        # one decoding step of one request: sigmoid scores with a balancing bias, latency only
        _route("route_1_decode", 1, 256, 8, "sigmoid", bias=True, scale=2.5, backward=False),
        # the router of a full training micro-batch of the 256-expert layer, with its load figures and its gradient
        _route("route_16k_train", 16384, 256, 8, "softmax"),
        # an odd number of tokens and experts, bf16 logits, some experts masked, weights not renormalised
        _route("route_5003_ragged", 5003, 60, 6, "softmax", renorm=False, dtype="bf16", masked=0.05),
        # balancing bias over a long micro-batch
        _route("route_32k_bias", 32768, 128, 8, "sigmoid", bias=True, scale=2.5),
        # the benchmark's smallest layer, two tokens: launches count
        _few("few_2_small", "bf16", 2, 1024, 512, 8, 2),
        # one token through one rank's share of the 256-expert layer: eight experts' weights are read
        _few("few_1_large", "bf16", 1, 7168, 2048, 32, 8),
        # an ordinary decoding batch, every expert touched by a few tokens
        _few("few_24_bf16", "bf16", 24, 5120, 1408, 64, 6),
        # the same kind of step with MXFP8 routed weights on one of two ranks, a padded batch and the clamped SwiGLU
        _few("few_48_mxfp8", "mxfp8", 48, 4096, 1536, 64, 8, ranks=2, limit=7.0, padded=0.25),
        # a full decoding batch of the large layer: all weights once
        _few("few_200_large", "bf16", 200, 7168, 2048, 32, 8),
        # a short micro-batch's activations, an odd row count
        _packed("restore_1031", "restore", 1031, 1024),
        # gate and up of an ordinary micro-batch
        _packed("swiglu8_25k", "swiglu8", 25088, 1408, limit=7.0),
        # one rank's share of the large layer: gate and up of all its routed rows
        _packed("swiglu8_135k", "swiglu8", 135168, 2048),
    ]


def _log_int(rng, low, high, step=1):
    """A multiple of `step` in [low, high], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + step)))
    return min(max(int(v) // step * step, low), high)


def draw(rng):
    op = rng.choice(["route", "few", "few", "restore", "swiglu8"])
    if op == "route":
        score = rng.choice(["softmax", "sigmoid"])
        experts = _log_int(rng, 8, 512)
        case = _route("", _log_int(rng, 1, 32768), experts, rng.randint(1, 8), score, bias=score == "sigmoid" and rng.random() < 0.7,
                      renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["fp32", "bf16"]),
                      masked=rng.choice([0.0, 0.0, 0.1]), backward=rng.random() < 0.8)
        case["tokens"] = min(case["tokens"], 32768 * 128 // experts)
    elif op == "few":
        hidden, inter = _log_int(rng, 1024, 7168, 256), _log_int(rng, 512, 2048, 128)
        experts = _log_int(rng, 8, 128)
        while experts > 8 and experts * hidden * inter > 32 * 7168 * 2048:
            experts -= 1
        case = _few("", rng.choice(["bf16", "bf16", "mxfp8"]), _log_int(rng, 1, 256), hidden, inter, experts, rng.randint(1, 8),
                    ranks=rng.choice([1, 1, 2, 4]), shared=rng.random() < 0.75, limit=rng.choice([0.0, 7.0]), padded=rng.choice([0.0, 0.0, 0.2]))
        while case["tokens"] * (case["topk"] + 1) * hidden * inter > 200 * 9 * 7168 * 2048:
            case["tokens"] -= 1
    else:
        cols = _log_int(rng, 512, 7168, 128)
        case = _packed("", op, _log_int(rng, 256, 135168), cols, limit=rng.choice([0.0, 7.0]) if op == "swiglu8" else 0.0)
        case["rows"] = min(case["rows"], 135168 * 2048 // cols)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------- inputs
def _mxfp8(w):
    """bf16 [E, M, N] -> E4M3 values and one power-of-two scale byte per 32 of N, in tiles of [M/128, N/128, 32, 16] (rows i of a
    128 x 128 tile at [i % 32], the four scales of row i at [4 * (i // 32)])."""
    E, M, N = w.shape
    v = w.float().view(E * M, N // 32, 32)
    scale = (v.abs().amax(-1) * 0.002232142857).clamp_min(1e-12)
    mantissa, exponent = torch.frexp(scale)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent)
    q = torch.ldexp(v, -exponent[:, :, None]).view(E, M, N).to(torch.float8_e4m3fn)
    tiles = (exponent + 127).to(torch.uint8).view(E * M // 128, 4, 32, N // 128, 4).permute(0, 3, 2, 1, 4)
    return q, tiles.reshape(E * M // 128, N // 128, 32, 16).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device=dev).normal_(0.0, std, generator=gen)

    s = {"case": case}
    if case["op"] == "route":
        T, E, K = case["tokens"], case["experts"], case["topk"]
        logits = normal(T, E, std=1.0, dtype=torch.float32) + normal(E, std=0.5, dtype=torch.float32)
        if case["masked"]:
            logits = logits.masked_fill(torch.rand(T, E, generator=gen, device=dev) < case["masked"], -math.inf)
            if T > 8:
                logits[T // 2] = -math.inf               # a row whose mask leaves nothing
        s["logits"] = logits.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        s["bias"] = normal(E, std=0.1, dtype=torch.float32) if case["bias"] else None
        s["d_weights"] = normal(T, K, std=1.0, dtype=torch.float32)
        s["d_score_sums"] = normal(E, std=1e-2, dtype=torch.float32)
    elif case["op"] == "few":
        T, H, I, E, K = (case[k] for k in ("tokens", "hidden", "inter", "experts", "topk"))
        s["x"] = normal(T, H, std=1.0)
        s["shared"] = tuple(normal(*d, std=0.02) for d in ((I, H), (I, H), (H, I))) if case["shared"] else (None, None, None)
        routed = tuple(normal(*d, std=0.02) for d in ((E, I, H), (E, I, H), (E, H, I)))
        s["routed"] = tuple(_mxfp8(w) for w in routed) if case["precision"] == "mxfp8" else routed
        logits = torch.randn(T, E * case["ranks"], generator=gen, device=dev)
        values, s["top_experts"] = torch.topk(logits, min(K, E * case["ranks"]), dim=1)
        weights = torch.softmax(values, -1)
        if case["padded"]:
            weights = weights * (torch.arange(T, device=dev) < T - int(T * case["padded"]))[:, None]
        s["router_weights"] = weights.contiguous()
        s["first_expert"] = E * (case["ranks"] - 1)
    else:
        n, c = case["rows"], case["cols"]
        # rows of different sizes, as tokens have
        s["x"] = normal(n, c, std=1.0) * torch.exp2(torch.randint(-2, 3, (n, 1), generator=gen, device=dev).float()).to(torch.bfloat16)
        if case["op"] == "swiglu8":
            s["up"], s["d_hidden"] = normal(n, c, std=2.0), normal(n, c, std=0.1)
            # router weights, and rows without one
            s["row_scale"] = (0.05 + 0.95 * torch.rand(n, generator=gen, device=dev)) * (torch.rand(n, generator=gen, device=dev) > 0.05)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_route(s):
    c, l = s["case"], s["logits"].float()
    K, scale = c["topk"], c["scale"]
    open_ = l > -math.inf
    if c["score"] == "softmax":
        key = l
        top = l.amax(-1, keepdim=True)
        e = torch.where(open_, torch.exp(l - top), 0.0)
        total = e.sum(-1, keepdim=True)
        score = torch.where(total > 0, e / total, 0.0)
    else:
        key = torch.sigmoid(l.double())
        if s["bias"] is not None:
            key = key + s["bias"].double()
        key = torch.where(open_, key, -math.inf).float() if s["bias"] is not None else l
        score = torch.where(open_, torch.sigmoid(l), 0.0)
    picked = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :K]      # ties: the lowest index first
    chosen = score.gather(1, picked)
    norm = chosen.sum(-1, keepdim=True)
    share = torch.where(norm > 0, chosen / norm, 0.0) if c["renorm"] else chosen
    out = {"top_experts": picked, "router_weights": share * scale}
    if not c["backward"]:
        return out
    out["tokens_per_expert"] = torch.zeros(c["experts"], dtype=torch.int32, device=l.device).index_add_(
        0, picked.reshape(-1), open_.gather(1, picked).reshape(-1).to(torch.int32))
    out["score_sums"] = score.sum(0)
    dw = s["d_weights"] * scale
    if c["renorm"]:
        # d share / d score: (dw - sum share * dw) / norm
        d_chosen = torch.where(norm > 0, (dw - (share * dw).sum(-1, keepdim=True)) / norm, 0.0)
    else:
        d_chosen = dw
    d_score = s["d_score_sums"].expand_as(score).scatter_add(1, picked, d_chosen)
    if c["score"] == "softmax":
        dl = score * (d_score - (score * d_score).sum(-1, keepdim=True))
    else:
        dl = d_score * score * (1.0 - score)
    out["d_logits"] = dl.to(s["logits"].dtype)
    return out


def _through_mxfp8(v):
    """What the E4M3 form with one power-of-two scale per 32 values holds of fp32 values."""
    b = v.reshape(-1, 32)
    scale = (b.abs().amax(-1, keepdim=True) * 0.002232142857).clamp_min(1e-12)
    mantissa, exponent = torch.frexp(scale)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent)
    return torch.ldexp(torch.ldexp(b, -exponent).to(torch.float8_e4m3fn).float(), exponent).view(v.shape)


def _scales(tiles, rows, cols):
    """Scale tiles -> fp32 factors [rows, cols / 32]."""
    exponent = tiles.view(rows // 128, cols // 128, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rows, cols // 32).to(torch.int32) - 127
    return torch.ldexp(torch.ones_like(exponent, dtype=torch.float32), exponent)


def _weights(w, experts=None):
    """Routed weights (of the experts named, or all) as fp32."""
    if isinstance(w, tuple):
        E, M, N = w[0].shape
        q, tiles = w[0], w[1].view(E, -1)
        if experts is not None:
            q, tiles, E = q.view(torch.uint8)[experts].view(torch.float8_e4m3fn), tiles[experts], experts.numel()
        return (q.float().view(E, M, N // 32, 32) * _scales(tiles, E * M, N).view(E, M, N // 32, 1)).view(E, M, N)
    return (w if experts is None else w[experts]).float()


def _swiglu(g, u, limit):
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g / (1.0 + torch.exp(-g)) * u


def _plain_few(s):
    c, x = s["case"], s["x"].float()
    T, H = x.shape
    E, limit = c["experts"], c["limit"]
    gate, up, down = s["routed"]
    keep = _through_mxfp8 if c["precision"] == "mxfp8" else lambda v: v
    e = s["top_experts"] - s["first_expert"]
    w = torch.where((e >= 0) & (e < E), s["router_weights"], 0.0)
    e = e.clamp(0, E - 1)
    xr = keep(x)
    if e.numel() < E:                                    # the routes' own weights, one product per route
        r = e.reshape(-1)
        xr = xr[:, None, :].expand(T, e.shape[1], H).reshape(-1, H, 1)
        h = _swiglu(torch.bmm(_weights(gate, r), xr), torch.bmm(_weights(up, r), xr), limit)
        y = (torch.bmm(_weights(down, r), keep(h.squeeze(-1)).unsqueeze(-1)).view(T, e.shape[1], H) * w[:, :, None]).sum(1)
    else:                                                # every expert over every token, weighted
        h = _swiglu(torch.matmul(xr, _weights(gate).mT), torch.matmul(xr, _weights(up).mT), limit)
        share = torch.zeros(T, E, device=x.device).scatter_add(1, e, w)
        y = (torch.bmm(keep(h), _weights(down).mT) * share.t()[:, :, None]).sum(0)
    if c["shared"]:
        g, u, d = (v.float() for v in s["shared"])
        y = y + _swiglu(x @ g.t(), x @ u.t(), limit) @ d.t()
    return y.to(torch.bfloat16)


def _plain_pack(x):
    """bf16 [n, c] -> whole numbers in [-127, 127], to the nearest, halves away from zero, and one fp32 scale per 128 values of a row.
    127 * b is exact in 32 bits and its quotient correctly rounded, so a half is a half."""
    b = x.float().unflatten(1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    some = top >= 2.0 ** -110
    q = torch.where(some, torch.floor(127.0 * b.abs() / top + 0.5) * b.sign(), 0.0)
    return q, torch.where(some, top / 127.0, 0.0)


def _plain_swiglu8(s):
    n, c = s["x"].shape
    limit = s["case"]["limit"]
    (gq, gs), (uq, us) = _plain_pack(s["x"]), _plain_pack(s["up"])
    g, u, dh = (gq * gs).view(n, c), (uq * us).view(n, c), s["d_hidden"].float()
    g_ok = u_ok = torch.ones((), dtype=torch.bool, device=g.device)
    if limit:
        g_ok, u_ok = g <= limit, u.abs() <= limit
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    sig = 1.0 / (1.0 + torch.exp(-g))
    silu = g * sig
    hidden = silu * u
    w = s["row_scale"]
    return {"d_gate": torch.where(g_ok, (silu * (1.0 - sig) + sig) * u * dh, 0.0).to(torch.bfloat16),
            "d_up": torch.where(u_ok, silu * dh, 0.0).to(torch.bfloat16), "hidden": hidden.to(torch.bfloat16),
            "row_grad": torch.where(w > 0, (dh * hidden).sum(-1) / w, 0.0)}


# ---------------------------------------------------------------------------------------------------- the framework's calls
def _mok():
    package = os.path.join(os.getcwd(), "mixture-of-kittens_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from mok import functional, ops
    return functional, ops


def _own_route(s):
    F, _ = _mok()
    c = s["case"]
    cfg = F.MoKRouterConfig(topk=c["topk"], score=c["score"], renormalize=c["renorm"], scale=c["scale"])
    r = F.route(cfg, s["logits"], s["bias"], balance=c["backward"])
    out = {"top_experts": r.top_experts, "router_weights": r.router_weights}
    if c["backward"]:
        out |= {"tokens_per_expert": r.tokens_per_expert, "score_sums": r.score_sums,
                "d_logits": F.route_backward(cfg, s["logits"], r, s["d_weights"], s["d_score_sums"])}
    return out


def _own_few(s):
    F, _ = _mok()
    return F.forward_few_tokens(s["x"], s["top_experts"], s["router_weights"], *s["shared"], *s["routed"], s["case"]["limit"] or None,
                                first_expert=s["first_expert"])


def _own_swiglu8(s):
    _, ops = _mok()
    gate, up = ops.pack_rows(s["x"]), ops.pack_rows(s["up"])
    d_gate, d_up, hidden, row_grad = ops.swiglu_bwd_packed(*gate, *up, s["d_hidden"], s["case"]["limit"] or None, s["row_scale"])
    return {"d_gate": d_gate, "d_up": d_up, "hidden": hidden, "row_grad": row_grad}


def run(state):
    op = state["case"]["op"]
    if op == "route":
        return _own_route(state) if own else _plain_route(state)
    if op == "few":
        return _own_few(state) if own else _plain_few(state)
    if op == "swiglu8":
        return _own_swiglu8(state) if own else _plain_swiglu8(state)
    if own:
        _, ops = _mok()
        return ops.unpack_rows(*ops.pack_rows(state["x"]))
    q, scale = _plain_pack(state["x"])
    return (q * scale).flatten(1).to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "route":
        T, E, K = case["tokens"], case["experts"], case["topk"]
        size = 2 if case["dtype"] == "bf16" else 4
        data, flops = T * E * size + 12 * T * K + (4 * E if case["bias"] else 0), 4 * T * E
        if case["backward"]:                             # logits again, their gradient; d_weights, the picks; load figures
            data, flops = data + 2 * T * E * size + 12 * T * K + 12 * E, flops + 8 * T * E
        return {"bytes": data, "flops": flops}
    if case["op"] == "few":
        T, H, I, E, K = (case[k] for k in ("tokens", "hidden", "inter", "experts", "topk"))
        live = T - int(T * case["padded"])
        K = min(K, E * case["ranks"])
        touched = E * (1.0 - (1.0 - K / (E * case["ranks"])) ** live)      # experts that have a token, on average
        size = 33 / 32 if case["precision"] == "mxfp8" else 2
        data = 3 * H * I * touched * size + 4 * T * H + 12 * T * K
        rows = live * K / case["ranks"]
        if case["shared"]:
            data, rows = data + 6 * H * I, rows + T
        return {"bytes": data, "flops": 6 * H * I * rows}
    n, c = case["rows"], case["cols"]
    kept = 1 + 4 / BLOCK
    if case["op"] == "restore":                          # bf16 in, packed out; packed in, bf16 out
        return {"bytes": n * c * (4 + 2 * kept), "flops": 4 * n * c}
    return {"bytes": n * c * (4 + 4 * kept + 2 + 6) + 8 * n, "flops": 30 * n * c}


# ---------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_route(s):
    c, l = s["case"], s["logits"].double()
    E, K = c["experts"], c["topk"]
    # the picks go by whole comparisons: of the logits themselves, or of the biased scores as 32-bit numbers
    order = 1.0 / (1.0 + torch.exp(-l))
    order = (order + s["bias"].double()).float().double() if s["bias"] is not None else l
    order = torch.where(torch.isneginf(l), -math.inf, order)
    picked = torch.argsort(order, dim=1, descending=True, stable=True)[:, :K]
    mask = torch.zeros_like(l).scatter_(1, picked, 1.0) * ~torch.isneginf(l)
    if c["score"] == "softmax":
        log_total = torch.logsumexp(l, 1, keepdim=True)
        score = torch.where(torch.isneginf(l), 0.0, torch.exp(l - torch.where(torch.isneginf(log_total), 0.0, log_total)))
    else:
        score = 1.0 / (1.0 + torch.exp(-l))
    norm = (score * mask).sum(1, keepdim=True)
    norm = torch.where(norm > 0, norm, 1.0)
    full = score * mask / norm if c["renorm"] else score * mask           # weights before `scale`, laid over all experts
    out = {"top_experts": None, "router_weights": full.gather(1, picked) * c["scale"]}
    if not c["backward"]:
        return out
    out |= {"tokens_per_expert": None, "score_sums": score.sum(0)}
    d = torch.zeros_like(l).scatter_(1, picked, s["d_weights"].double() * c["scale"]) * mask
    if c["renorm"]:
        d = mask * (d - (d * full).sum(1, keepdim=True)) / norm
    d = d + s["d_score_sums"].double()
    out["d_logits"] = score * (d - (d * score).sum(1, keepdim=True)) if c["score"] == "softmax" else score * (1.0 - score) * d
    return out


def _exact_few(s):
    c, x = s["case"], s["x"].double()
    limit, mx = c["limit"], c["precision"] == "mxfp8"

    def held(v):                                         # E4M3 with a power-of-two scale per 32 values, of 64-bit values
        if not mx:
            return v
        b = v.unflatten(-1, (-1, 32))
        scale = torch.exp2(torch.ceil(torch.log2((b.abs().amax(-1, keepdim=True) * 0.002232142857).clamp_min(1e-12))))
        return ((b / scale).float().to(torch.float8_e4m3fn).double() * scale).flatten(-2)

    def matrix(w, e):
        if not mx:
            return w[e].double()
        q, tiles = w[0][e], w[1].view(w[0].shape[0], -1, w[0].shape[2] // 128, 32, 4, 4)[e]
        exponent = tiles.permute(0, 3, 2, 1, 4).reshape(q.shape[0], -1).double() - 127.0
        return q.double() * torch.exp2(exponent).repeat_interleave(32, 1)

    def expert(v, g, u, d, hold):
        a, b = v @ g.t(), v @ u.t()
        if limit:
            a, b = torch.clamp(a, max=limit), torch.clamp(b, -limit, limit)
        return hold(a * torch.sigmoid(a) * b) @ d.t()

    y = torch.zeros_like(x)
    if c["shared"]:
        y += expert(x, *(w.double() for w in s["shared"]), lambda v: v)
    for e in range(c["experts"]):
        share = (s["router_weights"].double() * (s["top_experts"] == s["first_expert"] + e)).sum(1)
        rows = torch.nonzero(share).flatten()
        if rows.numel():
            y[rows] += share[rows, None] * expert(held(x[rows]), *(matrix(w, e) for w in s["routed"]), held)
    return y


def _exact_pack(x):
    b = x.double().unflatten(1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    steps = torch.floor((b.abs() * 254.0 + top) / (2.0 * torch.where(top > 0, top, 1.0)))      # floor(127 |b| / top + 1 / 2)
    return (torch.copysign(steps, b) * top / 127.0).flatten(1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s)
    if case["op"] == "few":
        return _exact_few(s)
    g = _exact_pack(s["x"])
    if case["op"] == "restore":
        return g
    u, dh, w = _exact_pack(s["up"]), s["d_hidden"].double(), s["row_scale"].double()
    inside_g = torch.ones_like(g) if not case["limit"] else (g <= case["limit"]).double()
    inside_u = torch.ones_like(u) if not case["limit"] else (u.abs() <= case["limit"]).double()
    if case["limit"]:
        g, u = g.clamp(max=case["limit"]), u.clamp(-case["limit"], case["limit"])
    sig = torch.sigmoid(g)
    hidden = g * sig * u
    inverse = torch.where(w > 0, 1.0 / w, 0.0)
    return {"d_gate": inside_g * sig * (1.0 + g * (1.0 - sig)) * u * dh, "d_up": inside_u * g * sig * dh, "hidden": hidden,
            "row_grad": (dh * hidden).sum(1) * inverse}
