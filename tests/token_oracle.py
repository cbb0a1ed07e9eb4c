"""64-bit definitions of the token operators for their tests, each with how far a correct kernel may be off, element by element.

Bounds count: half a step (u = eps / 2 of the type) for every rounding to 16 bits, 2^-24 for every float32 operation of a sum of n terms
(n * 2^-24 * the sum of magnitudes), and what an error of the arguments does to sin, cos and exp2."""
import math

import torch

F32 = 2.0 ** -24
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: F32}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half of the smallest step near zero


def visible(B, Tk, lengths, mask, device="cpu"):
    seen = torch.ones((B, Tk), dtype=torch.bool, device=device)
    if lengths is not None:
        seen = seen & (torch.arange(Tk, device=device)[None] < lengths.to(device)[:, None])
    return seen if mask is None else seen & mask.to(device)


def attention(q, k, v, lengths=None, mask=None, scale=None, dout=None):
    """-> dict of (value, allowance) pairs: out, lse and with dout dq, dk, dv (and "sums": two parts of allowances); tensors as the operator takes them"""
    B, Tq, H, D = q.shape
    Tk, K = k.shape[1:3]
    G, u, tiny, dtype = H // K, UNIT[q.dtype], TINY[q.dtype], torch.float64
    scale = 1 / math.sqrt(D) if scale is None else scale
    seen = visible(B, Tk, lengths, mask, q.device)[:, None, None, :]
    heads = lambda t: t.to(dtype).transpose(1, 2).contiguous()  # noqa: E731  (B, heads, T, D)
    hide = ~seen[:, 0, 0, :, None, None]
    q_, k_, v_ = heads(q), heads(k.masked_fill(hide, 0)), heads(v.masked_fill(hide, 0))
    k_, v_ = k_.repeat_interleave(G, 1), v_.repeat_interleave(G, 1)
    kt, vt = k_.transpose(2, 3).contiguous(), v_.transpose(2, 3).contiguous()
    s = (q_ @ kt * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    some = seen.any(-1).expand(B, H, Tq) if Tk else torch.zeros((B, H, Tq), dtype=torch.bool, device=q.device)
    w = torch.where(some[..., None], (s - lse.masked_fill(~some, 0)[..., None]).exp(), torch.zeros_like(s)) if Tk else s
    out = w @ v_
    # scores: a float32 dot product of D terms, then c s - m in base 2, each |s| 2^-23 off at most; the same for the maximum's side
    mag = (q_.abs() @ kt.abs() * scale).masked_fill(~seen, 0)
    es = mag.amax(-1, keepdim=True) * (D + 8) * 2 * F32 if Tk else torch.zeros_like(out[..., :1])
    near = 2 * es + (Tk + 64) * F32  # relative: a weight (2 es) and the sums that it is in
    lost = 2.0 ** -31 * Tk if q.dtype == torch.float16 else 0.0  # weights below fp16's range
    wv = w @ v_.abs()
    top = v_.abs().amax(2, keepdim=True) if Tk else torch.zeros_like(out[:, :, :1])
    e_out = wv * (u + near) + lost * top  # before its own rounding
    got = {"out": (out, e_out + u * (out.abs() + e_out) + tiny), "lse": (lse, (es + (Tk + 64) * F32)[..., 0] + 4 * F32 * lse.abs().nan_to_num(0, 0, 0))}
    if dout is not None:
        do = heads(dout)
        dw = do @ vt
        delta = (do * out).sum(-1, keepdim=True)
        ds = w * (dw - delta)
        # delta comes from the rounded output; dw and delta are float32 dot products of D terms
        e_delta = (do.abs() * (e_out + u * out.abs() + tiny)).sum(-1, keepdim=True)
        e_dw = (do.abs() @ vt.abs() + (do.abs() * out.abs()).sum(-1, keepdim=True)) * (D + 8) * F32
        e_ds = ds.abs() * (u + near) + w * (e_delta + e_dw)
        share = lambda t: t.reshape(B, K, G, Tk, D).sum(2)  # noqa: E731
        wt, dst = w.transpose(2, 3).contiguous(), ds.transpose(2, 3).contiguous()
        ewt, edst = (w * (u + near)).transpose(2, 3).contiguous(), e_ds.transpose(2, 3).contiguous()
        rows = (Tq * G + 64) * F32
        dv, e_dv = share(wt @ do), share(ewt @ do.abs() + rows * (wt @ do.abs()))
        dk, e_dk = share(dst @ q_) * scale, share(edst @ q_.abs() + rows * (dst.abs() @ q_.abs())) * scale
        dq, e_dq = ds @ k_ * scale, (e_ds @ k_.abs() + (Tk + 64) * F32 * (ds.abs() @ k_.abs())) * scale
        if q.dtype == torch.float16 and Tq and Tk:
            # 2^-38 of 1 for w, 2^-37 of a column's largest ds (attention_bwd.hip): a step's half, times the other operand
            e_dv = e_dv + 2.0 ** -38 * share(do.abs().sum(2, keepdim=True).expand(B, H, Tk, D))
            e_dk = e_dk + 2.0 ** -37 * share(ds.abs().amax(2)[..., None] * q_.abs().sum(2, keepdim=True)) * scale
            e_dq = e_dq + 2.0 ** -37 * ds.abs().amax(-1, keepdim=True) * k_.abs().sum(2, keepdim=True) * scale
        for name, x, e in (("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv)):
            got[name] = (x, e + u * (x.abs() + e) + tiny)
        # of the allowances of dq and dk, what the float32 sums in dw - delta alone make: all that is left where one key has the whole weight
        got["sums"] = ((w * e_dw) @ k_.abs() * scale, share((w * e_dw).transpose(2, 3).contiguous() @ q_.abs()) * scale)
    return {n: (a.transpose(1, 2), b.transpose(1, 2)) if a.dim() == 4 else (a, b) for n, (a, b) in got.items()}


def rotary(x, positions, sections, theta=10000.0, ladder="axis", interleaved=False, inverse=False):
    """-> (value, allowance)"""
    P = sum(sections)
    power = [i / n for n in sections for i in range(n)] if ladder == "axis" else [j / P for j in range(P)]
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    freq = torch.tensor([theta ** -p for p in power], dtype=torch.float64, device=x.device)
    angle = positions.double()[..., axis] * freq * (-1 if inverse else 1)
    c, s = angle.cos()[..., None, :], angle.sin()[..., None, :]
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    i, j = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    a, b = x.double()[..., i], x.double()[..., j]
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    size[..., i] = size[..., j] = a.abs() + b.abs()
    # the fraction of a turn is rounded to float32 (2 pi 2^-25), sine and cosine are 2 units off at most (2^-23), three operations; the
    # 64-bit angle itself is 2^-51 of its size off
    far = float(angle.abs().max()) * 2.0 ** -51 if angle.numel() else 0.0
    return y, size * (2 * math.pi * 2.0 ** -25 + 2.0 ** -22 + 3 * F32 + far) + UNIT[x.dtype] * (y.abs() * 1.001) + TINY[x.dtype]


def adamw(p, g, m, v, w=None, step=1, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01):
    """-> dict of (value, allowance) of one step; w: the running maximum (amsgrad)"""
    b1, b2 = betas
    P, g, m, v = p.double(), g.double(), m.double(), v.double()
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    # two products, a sum and constants that are themselves rounded: 4 roundings of each term
    e_m, e_v = 4 * F32 * (b1 * m.abs() + (1 - b1) * g.abs()), 5 * F32 * v1
    got = {"exp_avg": (m1, e_m), "exp_avg_sq": (v1, e_v)}
    u = v1
    if w is not None:
        u = torch.maximum(w.double(), v1)
        got["max_exp_avg_sq"] = (u, e_v)
    c1, c2 = 1 - b1 ** step, math.sqrt(1 - b2 ** step)
    root = u.sqrt() / c2 + eps
    move = lr / c1 * m1 / root
    x = P * (1 - lr * weight_decay) - move
    # the move: m1's error, root half of u's relative 5 plus 4 more roundings, the quotient and its factors 5
    e = lr / c1 * e_m / root + move.abs() * 12 * F32 + 4 * F32 * (P.abs() + move.abs())
    got["param"] = (x, e + UNIT[p.dtype] * (x.abs() + e) + TINY[p.dtype])
    return got


def worst(got, pair):
    """The largest |got - value| / allowance (at most 1 is right); places where value is not finite have to be equal."""
    value, allowed = pair
    assert got.shape == value.shape, (got.shape, value.shape)
    got, value, allowed = got.double(), value, allowed.expand_as(value) if allowed.shape != value.shape else allowed
    fine = torch.isfinite(value)
    assert torch.equal(got[~fine].nan_to_num(7.0), value[~fine].nan_to_num(7.0)), "non-finite places differ"
    off = (got - value).abs()[fine]
    allowed = allowed[fine]
    if not off.numel():
        return 0.0
    assert torch.isfinite(off).all(), "non-finite results"
    return float((off / allowed.clamp_min(1e-300)).max())
