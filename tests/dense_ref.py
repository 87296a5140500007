"""Plain 64-bit forms of the dense attention operators, with bounds on what a kernel that rounds
as documented may be off by.

A value rounded to b bits is off by at most half a step (bf16 2^-8, fp32 2^-24 relative); sums of
n products in fp32 by n steps of 2^-24 of the sum of magnitudes.  The bounds follow those
roundings through the formulas, first order, element by element.
"""

import math

import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def lens_to_cu(lens, device):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def attention(q, k, v, lens_q, lens_k, heads, kv, causal, scale=None, dout=None, dlse=None,
              seen=None):
    """out, lse (, dq, dk, dv) of packed sequences in float64 and a bound on each result's error.
    ``seen(s, lq, lk)``: mask of sequence s in place of the causal or full one."""
    dt, dev = q.dtype, q.device
    hd = q.shape[-1] // heads
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    f = dict(dtype=torch.float64, device=dev)
    N, M, grp = q.shape[0], k.shape[0], heads // kv
    out, lse = torch.zeros(q.shape, **f), torch.full((N, heads), -math.inf, **f)
    eo, el = torch.zeros_like(out), torch.zeros_like(lse)
    grads = [torch.zeros(t.shape, **f) for t in (q, k, v)] if dout is not None else None
    errs = [torch.zeros(t.shape, **f) for t in (q, k, v)] if dout is not None else None
    h = HALF[dt]
    a0 = b0 = 0
    for s, (a, b) in enumerate(zip(lens_q, lens_k)):
        R, C = slice(a0, a0 + a), slice(b0, b0 + b)
        a0, b0 = a0 + a, b0 + b
        if a == 0 or b == 0:
            continue
        if seen is not None:
            m = seen(s, a, b)
        else:
            m = torch.ones(a, b, dtype=torch.bool, device=dev)
            m = m.tril(b - a) if causal else m
        for hh in range(heads):
            c, ck = slice(hh * hd, hh * hd + hd), slice(hh // grp * hd, hh // grp * hd + hd)
            Q, K, V = q[R, c].double(), k[C, ck].double(), v[C, ck].double()
            x = Q @ K.t() * scale
            mag = Q.abs() @ K.abs().t() * scale
            x = x.masked_fill(~m, -math.inf)
            top = x.amax(1, keepdim=True)
            top = torch.where(top == -math.inf, torch.zeros_like(top), top)
            e = torch.exp(x - top)
            l = e.sum(1, keepdim=True)
            ok = (l > 0).double()
            p = torch.where(l > 0, e / l.clamp_min(1e-300), torch.zeros_like(e))
            O = p @ V
            out[R, c] = O
            lse[R, hh] = torch.where(l > 0, top + torch.log(l), torch.full_like(l, -math.inf))[:, 0]
            # score: hd products and the scale; exponent: two more roundings of its argument and
            # one of its value; sums of b terms
            es = ((hd + 4) * U * mag).masked_fill(~m, 0.0).amax(1, keepdim=True)
            es = es + 4 * U * (top.abs() + 16)  # arguments up to the largest score, 2^8 above it
            # es: a bound on the relative error of every weight and of their sum
            rel = 2 * es + (b + 64) * U
            if dt == torch.bfloat16:
                rel = rel + h  # the weights are rounded once
            pv = p @ V.abs()
            eo[R, c] = ok * (rel * pv + h * O.abs())
            el[R, hh] = (ok * (es + (b + 64) * U + 4 * U * (top.abs() + 16)))[:, 0]
            if dout is None:
                continue
            G = dout[R, c].double()
            dp = G @ V.t()
            delta = (G * O).sum(1, keepdim=True)
            if dlse is not None:
                delta = delta - dlse[R, hh].double()[:, None]
            ds = p * (dp - delta)
            grads[0][R, c] = ds @ K * scale
            grads[1][C, ck] += ds.t() @ Q * scale
            grads[2][C, ck] += p.t() @ G
            # delta: from the rounded out; dp: hd products; then ds rounded
            ed = (G.abs() * eo[R, c]).sum(1, keepdim=True) + (hd + 2) * U * (
                G.abs() @ V.abs().t() + (G.abs() * O.abs()).sum(1, keepdim=True) +
                (0 if dlse is None else dlse[R, hh].double().abs()[:, None]))
            ep = 2 * es + (b + 64) * U + 4 * U * lse[R, hh].abs().nan_to_num(0.0, 0.0, 0.0)[:, None]
            eds = p * ed + ep * ds.abs() + (h if dt == torch.bfloat16 else 4 * U) * ds.abs()
            errs[0][R, c] += (eds + (b + 8) * U * ds.abs()) @ K.abs() * scale
            errs[1][C, ck] += ((eds + (a * grp + 8) * U * ds.abs()).t() @ Q.abs()) * scale
            errs[2][C, ck] += ((ep + (h if dt == torch.bfloat16 else 0.0) +
                                (a * grp + 8) * U) * p).t() @ G.abs()
    if dout is None:
        return (out, lse), (eo, el)
    errs = [e + h * g.abs() for e, g in zip(errs, grads)]
    return (out, lse, *grads), (eo, el, *errs)


def assert_within(got, want, err, what, slack=1e-30):
    """Every element within its bound (times 1.01 for second-order terms), and finite as wanted."""
    g, w = got.double(), want.double()
    same = (g == w) | (g.isnan() & w.isnan())
    d = torch.where(same, torch.zeros_like(w), (g - w).abs())
    over = ~(d <= 1.01 * err + slack)
    if over.any():
        i = int(torch.where(over, (d / (err + 1e-30)).nan_to_num(1e30), 0.0 * d).argmax())
        raise AssertionError(
            f"{what}: {int(over.sum())} of {over.numel()} beyond their bound; worst at {i}: got "
            f"{float(g.flatten()[i])}, want {float(w.flatten()[i])}, bound {float(err.flatten()[i])}")


# ---------------------------------------------------------------------------
# rotation, norm
# ---------------------------------------------------------------------------

def turn(x, pos, axes, theta, interleaved, sign=1.0):
    """x [..., N, heads, hd] float64 turned by pos [..., N, axes]."""
    y = x.clone()
    at = 0
    for a, d in enumerate(axes):
        i = torch.arange(d // 2, device=x.device)
        ang = sign * pos[..., a].double()[..., None, None] * theta ** (-2.0 * i.double() / max(d, 1))
        u, w = (at + 2 * i, at + 2 * i + 1) if interleaved else (at + i, at + i + d // 2)
        c, s = ang.cos(), ang.sin()
        y[..., u] = x[..., u] * c - x[..., w] * s
        y[..., w] = x[..., u] * s + x[..., w] * c
        at += d
    return y


def turn_mag(x, axes, interleaved):
    """|a| + |b| of each channel's pair (the channel itself where it passes through)."""
    y = x.abs().clone()
    at = 0
    for d in axes:
        i = torch.arange(d // 2, device=x.device)
        u, w = (at + 2 * i, at + 2 * i + 1) if interleaved else (at + i, at + i + d // 2)
        y[..., u] = y[..., w] = x[..., u].abs() + x[..., w].abs()
        at += d
    return y


def norm_rope(x, w, pos, heads, axes, theta, eps, interleaved, dy=None, norm=True):
    """y (, dx, dw) in float64 and bounds.  Steps of 2^-24 of the magnitudes: the turn's cosine
    and sine 8 (angle, function), its products and sum 3; the norm's mean square hd / 8 + 16 (a
    lane's sum, then a tree), the root, two products 6."""
    hd, h = x.shape[-1] // heads, HALF[x.dtype]
    n = (11 + (hd / 8 + 24 if norm else 0)) * U
    X = x.double().unflatten(-1, (heads, hd))
    r = (X.square().mean(-1, keepdim=True) + eps).rsqrt() if norm else torch.ones_like(X[..., :1])
    W = torch.ones(hd, dtype=torch.float64, device=x.device) if w is None else w.double()
    Y = turn(X * r * W, pos, axes, theta, interleaved)
    ey = h * Y.abs() + n * turn_mag(X * r * W, axes, interleaved)
    if dy is None:
        return (Y.flatten(-2),), (ey.flatten(-2),)
    G = dy.double().unflatten(-1, (heads, hd))
    g, gm = turn(G, pos, axes, theta, interleaved, -1.0), turn_mag(G, axes, interleaved)
    if not norm:
        return (Y.flatten(-2), g.flatten(-2)), (ey.flatten(-2), (h * g.abs() + n * gm).flatten(-2))
    dims = tuple(range(X.dim() - 1))
    dw = (g * X * r).sum(dims)
    rows = X[..., 0].numel()
    edw = ((n + rows * U) * (gm * X.abs() * r)).sum(dims)
    dot = (g * W * X).mean(-1, keepdim=True)
    dx = r * (g * W) - X * r ** 3 * dot
    mag = r * gm * W.abs() + X.abs() * r ** 3 * (gm * W.abs() * X.abs()).mean(-1, keepdim=True)
    edx = h * dx.abs() + (4 * n) * mag
    return (Y.flatten(-2), dx.flatten(-2), dw), (ey.flatten(-2), edx.flatten(-2), edw)
