"""Plain implementations in 64 bits of the operators around the layer (router, few tokens, 8-bit activations), with the
error bounds that the tests hold the kernels to.  Every bound counts roundings: U32 for one of fp32 (half a step), U16 for one of bf16."""
import torch

U32 = torch.finfo(torch.float32).eps / 2
U16 = torch.finfo(torch.bfloat16).eps / 2


# ------------------------------------------------------------------------------------------------------------- router
def route(logits, topk, score, bias=None, renormalize=True, scale=1.0):
    """(top_experts, weights, tokens_per_expert, score_sums, s, mask of open picks) in 64 bits."""
    l = logits.double()
    l = torch.where(torch.isnan(l), -torch.inf, l).clamp(max=torch.finfo(torch.float32).max)
    closed = torch.isneginf(l)
    if score == "softmax":
        key = l
        s = torch.softmax(torch.where(closed.all(1, keepdim=True), 0.0, l), 1) * ~closed
    else:
        s = torch.sigmoid(l)
        key = l if bias is None else (s + bias.double()).float().double()
    key = torch.where(closed, -torch.inf, key)
    picked = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :topk]
    chosen = s.gather(1, picked)
    norm = chosen.sum(1, keepdim=True)
    share = torch.where(norm > 0, chosen / torch.where(norm > 0, norm, 1.0), 0.0) if renormalize else chosen
    open_picks = ~closed.gather(1, picked)
    counts = torch.zeros(l.shape[1], dtype=torch.int64, device=l.device).index_add_(0, picked.reshape(-1), open_picks.reshape(-1).long())
    return picked, share * scale, counts, s.sum(0), s, open_picks


def route_bwd(logits, picked, d_weights, d_sums, score, renormalize, scale):
    """The gradient of the logits by autograd in 64 bits, from the scores' definition."""
    l = logits.double()
    l = torch.where(torch.isnan(l), -torch.inf, l).clamp(max=torch.finfo(torch.float32).max)
    closed = torch.isneginf(l)
    top = l.amax(1, keepdim=True)
    top = torch.where(torch.isneginf(top), 0.0, top)
    leaf = torch.where(closed, top, l).requires_grad_(True)      # (closed experts are left out below; any number of the row's size will do)
    if score == "softmax":
        e = torch.exp(leaf - top) * ~closed
        total = e.sum(1, keepdim=True)
        s = e / torch.where(total > 0, total, 1.0)
    else:
        s = torch.sigmoid(leaf) * ~closed
    chosen = s.gather(1, picked)
    norm = chosen.sum(1, keepdim=True)
    w = (chosen / torch.where(norm > 0, norm, 1.0) if renormalize else chosen) * scale
    loss = (w * d_weights.double()).sum()
    if d_sums is not None:
        loss = loss + (s.sum(0) * d_sums.double()).sum()
    return torch.autograd.grad(loss, leaf)[0] * ~closed


# ------------------------------------------------------------------------------------------------------------- few tokens
def _e4m3(v):
    return v.to(torch.float32).to(torch.float8_e4m3fn).double()


def mx_scale(v):
    """Power-of-two scale of each 32 values along the last axis, [.., n / 32, 1]."""
    top = v.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).float()
    scale = torch.clamp(top * 0.002232142857, min=1e-12)
    m, e = torch.frexp(scale)
    return torch.exp2(torch.where(m == 0.5, e - 1, e).double())


def mx_hold(v, scale=None):
    """What E4M3 with that scale holds of 64-bit values."""
    scale = mx_scale(v) if scale is None else scale
    return (_e4m3(v.unflatten(-1, (-1, 32)) / scale) * scale).flatten(-2)


def mx_dequantize(q, tiles):
    """E4M3 [E, M, N] and scale tiles [E * M / 128, N / 128, 32, 16] -> 64 bits."""
    E, M, N = q.shape
    exponent = tiles.view(E * M // 128, N // 128, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(E, M, N // 32, 1).double() - 127.0
    return (q.double().view(E, M, N // 32, 32) * torch.exp2(exponent)).view(E, M, N)


def _silu(g):
    return g * torch.sigmoid(g)


def expert(x, wg, wu, wd, limit, mx):
    """One expert over rows x [n, H] (64 bits) -> (y [n, H], bound of what the kernel's y may be off before its last rounding).

    Sums of n products in fp32 are off by at most n roundings of the sum of their absolute values; a silu by a few roundings of
    itself and 1.1 times its argument's error (|silu'| < 1.1); hidden is rounded once: to bf16, or to E4M3, where it may fall on
    either side of a rounding border that lies inside its own error."""
    H, I = wg.shape[1], wg.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = (H + 4) * U32 * (x.abs() @ wg.abs().t()), (H + 4) * U32 * (x.abs() @ wu.abs().t())
    if limit is not None:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    s = _silu(g)
    h = s * u
    eh = (1.1 * eg + 16 * U32 * s.abs()) * u.abs() + s.abs() * eu + 1.1 * eg * eu + 4 * U32 * h.abs()
    if mx:
        # the block's largest value, and with it the scale, is known to within its error too
        held = mx_hold(h)
        wide = (h.abs() + eh).unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)
        slim = (h.abs() - eh).clamp_min(0.0).unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)
        eh = torch.stack([(mx_hold(v, mx_scale(top)) - held).abs() for v in (h - eh, h + eh) for top in (slim, wide)]).amax(0)
        h = held
    else:
        eh = eh + U16 * (h.abs() + eh)
    y = h @ wd.t()
    return y, eh @ wd.abs().t() + (I + 4) * U32 * ((h.abs() + eh) @ wd.abs().t())


def few_tokens(x, top_experts, weights, shared, routed, limit=None, first=0, mx=False):
    """(y, bound) in 64 bits; `routed`: bf16 [E, ..] weights, or (E4M3, tiles) pairs with `mx`."""
    x = x.double()
    wg, wu, wd = ((mx_dequantize(*w) if mx else w.double()) for w in routed)
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    if shared is not None:
        y, bound = expert(x, *(w.double() for w in shared), limit, False)
    xr = mx_hold(x) if mx else x
    for e in range(wg.shape[0]):
        share = weights.double() * (top_experts == first + e)
        rows = torch.nonzero(share.abs().sum(1)).flatten()
        if rows.numel() == 0:
            continue
        ye, be = expert(xr[rows], wg[e], wu[e], wd[e], limit, mx)
        for k in range(weights.shape[1]):                # an expert may be named twice
            w = share[rows, k, None]
            y[rows] += w * ye
            bound[rows] += w.abs() * (be + 3 * U32 * ye.abs())
    K = weights.shape[1]
    bound += (K + 2) * U32 * (y.abs() + bound)
    return y, bound + U16 * (y.abs() + bound)


# ------------------------------------------------------------------------------------------------------------- 8-bit activations
def pack(x):
    """bf16 [n, c] -> (q int8, scales fp32 bits by one division, values in 64 bits)."""
    n, c = x.shape
    blocks = -(-c // 128)
    v = torch.zeros(n, blocks * 128, dtype=torch.float64, device=x.device)
    v[:, :c] = x.double()
    v = v.view(n, blocks, 128)
    top = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    some = (top >= 2.0 ** -110) & ~bad
    # floor(127 |v| / top + 1 / 2) as the quotient of whole multiples: halves are exact
    q = torch.where(some, torch.floor((254.0 * v.abs() + top) / (2.0 * torch.where(some, top, 1.0))), 0.0) * v.sign().nan_to_num()
    q = torch.where(bad, 0.0, q)
    scales = torch.where(some, (top / torch.full_like(top, 127.0)).float(), 0.0).masked_fill(bad, torch.nan)      # (by a tensor: by a number, torch multiplies by its reciprocal)
    values = (q * scales.double()).view(n, -1)[:, :c]
    return q.view(n, -1)[:, :c].to(torch.int8), scales.squeeze(-1).float(), values


def swiglu_bwd(g, u, dh, limit=None, row_scale=None):
    """d_gate, d_up, hidden, row_grad in 64 bits of 64-bit gate and up."""
    inside_g = inside_u = torch.ones_like(g, dtype=torch.bool)
    if limit is not None:
        inside_g, inside_u = ~(g > limit), ~(u.abs() > limit)
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    sig = torch.sigmoid(g)
    h = g * sig * u
    w = torch.ones(g.shape[0], dtype=torch.float64, device=g.device) if row_scale is None else row_scale.double()
    inv = torch.where(w > 0, 1.0 / torch.where(w > 0, w, 1.0), 0.0)
    return (torch.where(inside_g, sig * (1 + g * (1 - sig)) * u * dh, 0.0), torch.where(inside_u, g * sig * dh, 0.0), h,
            (dh * h).sum(1) * inv)
