"""Operators of dense attention layers: rotary positions with several axes, the norm of queries
and keys with that rotation, and attention over packed sequences with grouped heads.

``listed`` gives the fixed cases, ``draw`` another of the same ranges; ``prepare`` makes what a
program holds before the call, ``run`` is one pass (the plain form, or the framework's operators
where ``own`` is true), ``work`` its bytes and operations, ``exact`` the results in float64.
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _rope(name, T, H, W, heads, hd, dtype="bf16", B=1, interleaved=True, train=True):
    return {"name": name, "kind": "rope", "B": B, "T": T, "H": H, "W": W, "heads": heads,
            "kv_heads": 0, "head_dim": hd, "dtype": dtype, "interleaved": interleaved,
            "train": train, "far": 0}


def _norm(name, T, H, W, heads, kv, hd, dtype="bf16", B=1, interleaved=False, train=True, far=0):
    """far > 0: T tokens at positions below ``far`` on one axis (text) instead of a video grid."""
    return {"name": name, "kind": "norm", "B": B, "T": T, "H": H, "W": W, "heads": heads,
            "kv_heads": kv, "head_dim": hd, "dtype": dtype, "interleaved": interleaved,
            "train": train, "far": far}


def _attn(name, q_lens, k_lens, heads, kv, hd, causal, dtype="bf16", train=True):
    """Lengths of the packed sequences, joined by '+'; k_lens "" where they are the queries'."""
    return {"name": name, "kind": "attn", "q_lens": q_lens, "k_lens": k_lens, "heads": heads,
            "kv_heads": kv, "head_dim": hd, "causal": causal, "dtype": dtype, "train": train}


def listed():
    return [
        # a small fp32 model at inference, 2,048 video tokens: launches and latency count
        _rope("rope_small_fp32", 8, 16, 16, 4, 64, dtype="fp32", interleaved=False, train=False),
        # a training layer of 46,800 tokens on a grid that no tile divides
        _rope("rope_train_ragged_bf16", 13, 45, 80, 16, 96),
        # the newest token of 16 sequences, far along one axis: serving's latency
        _norm("norm_tokens_bf16", 16, 1, 1, 32, 8, 128, train=False, far=131072),
        # fp32 training, batch of two
        _norm("norm_train_fp32", 16, 32, 32, 8, 8, 64, dtype="fp32", B=2, interleaved=True),
        # a 256-frame clip in training
        _norm("norm_train_long_bf16", 64, 32, 32, 16, 16, 64),
        # one new token of one short sequence: latency
        _attn("attn_token_short_bf16", "1", "257", 16, 4, 64, True, train=False),
        # one new token each for 16 sequences whose caches hold 1 to 32,768 tokens
        _attn("attn_tokens_long_bf16", "+".join(["1"] * 16),
              "1+130+517+1024+2049+3000+4096+5003+6143+8192+9001+10240+12289+16384+20011+32768",
              32, 8, 128, True, train=False),
        # prompts of different lengths packed into one call, forward only
        _attn("attn_prompts_bf16", "1+37+0+311+700+1311+2053+4096", "", 32, 8, 128, True,
              train=False),
        # packed training sequences, causal, grouped heads
        _attn("attn_train_packed_bf16", "129+1000+2047+4500+5003", "", 16, 4, 128, True),
        # dense attention over one clip of 8,192 video tokens
        _attn("attn_train_clip_bf16", "8192", "", 16, 16, 64, False),
        # a small fp32 model's training layer, two clips of 2,048 tokens
        _attn("attn_train_small_fp32", "2048+2048", "", 4, 4, 64, False, dtype="fp32"),
        # a width of 1,280 over 16 heads: a head size that is no multiple of 32
        _attn("attn_train_hd80_bf16", "3375+721", "", 16, 16, 80, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    group = rng.choice([1, 1, 2, 3, 4, 8])
    kv = rng.choice([1, 2, 4, 5, 8, 16])
    return min(group, 32 // kv) * kv, kv


def _lens(ns):
    return [int(s) for s in ns.split("+")]


def _padded(q, k, heads):
    """Scores of the plain form, which pads every sequence to the longest."""
    return len(q) * max(q) * max(k) * heads


def draw(rng):
    """One more case: a rotation (with or without the norm) in four of ten, single tokens over
    caches in two, whole sequences in four."""
    u = rng.random()
    dtype = "bf16" if rng.random() < 0.7 else "fp32"
    if u < 0.4:
        B = rng.choice([1, 1, 2, 3])
        while True:
            T, H, W = _log_int(rng, 1, 64), _log_int(rng, 2, 64), _log_int(rng, 2, 96)
            heads, kv = _heads(rng)
            hd = rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 128, 128])
            if 2 ** 16 <= B * T * H * W * (heads + kv) * hd <= 2 ** 26:
                break
        inter, train = rng.random() < 0.5, rng.random() < 0.7
        if rng.random() < 0.4:
            c = _rope("", T, H, W, heads, hd, dtype, B, inter, train)
        elif rng.random() < 0.3:
            c = _norm("", T * H * W, 1, 1, heads, kv, hd, dtype, B, inter, train,
                      max(T * H * W, _log_int(rng, 1000, 1000000)))
        else:
            c = _norm("", T, H, W, heads, kv, hd, dtype, B, inter, train)
    else:
        hd = rng.choice([32, 64, 64, 80, 96, 128, 128])
        causal = rng.random() < 0.6
        while True:
            S = _log_int(rng, 1, 24)
            heads, kv = _heads(rng)
            if u < 0.6:
                top = _log_int(rng, 64, 32768)
                k = [_log_int(rng, 1, top) for _ in range(S)]
                q = [1] * S
                if 2 ** 14 <= sum(k) * kv * hd <= 2 ** 27 and _padded(q, k, kv) * hd <= 2 ** 28:
                    break
            else:
                top = _log_int(rng, 16, 6000)
                k = [rng.choice([0, 1, top]) if rng.random() < 0.2 else rng.randint(1, top)
                     for _ in range(S)]
                k[rng.randrange(S)] = top
                q = k
                cap = 2 ** 30 if dtype == "bf16" else 2 ** 28
                if 2 ** 14 <= _padded(q, k, heads) <= cap:
                    break
        text = "+".join(map(str, k))
        if u < 0.6:
            c = _attn("", "+".join(map(str, q)), text, heads, kv, hd, causal, dtype, False)
        else:
            c = _attn("", text, "", heads, kv, hd, causal, dtype, rng.random() < 0.7)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _axes(c):
    """Channels turned by time, height and width (all by one axis for text)."""
    hd = c["head_dim"]
    if c["far"]:
        return (hd,)
    side = 2 * (hd // 6)
    return (hd - 2 * side, side, side)


def _positions(c, g):
    if c["far"]:
        pos = torch.randint(0, c["far"], (c["B"], c["T"], 1), generator=g, device="cuda")
        return pos.to(torch.int32)
    t, h, w = (torch.arange(n, device="cuda", dtype=torch.int32) for n in (c["T"], c["H"], c["W"]))
    return torch.stack(torch.meshgrid(t, h, w, indexing="ij"), -1).reshape(-1, 3).contiguous()


def _qk_inputs(c, seed):
    """q, k (views of one fused projection's output), weights near one, positions and, for
    training, the gradients of both results."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, hd = _DT[c["dtype"]], c["head_dim"]
    B, N = c["B"], c["T"] * c["H"] * c["W"]
    nq, nk = c["heads"] * hd, c["kv_heads"] * hd

    def r(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std)

    fused = r(B, N, nq + 2 * nk, std=1.5).to(dt)
    q, k = fused[..., :nq], fused[..., nq:nq + nk]
    wq, wk = 1.0 + r(hd, std=0.1), 1.0 + r(hd, std=0.1)
    dq, dk = (r(B, N, n).to(dt) if c["train"] else None for n in (nq, nk))
    return q, k, wq, wk, _positions(c, g), dq, dk


def _attn_lens(c):
    q = _lens(c["q_lens"])
    return q, _lens(c["k_lens"]) if c["k_lens"] else q


def _attn_inputs(c, seed):
    """Queries and keys as after their norm (queries a little wider, so that weights differ)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, hd = _DT[c["dtype"]], c["head_dim"]
    ql, kl = _attn_lens(c)
    nq, nk = c["heads"] * hd, c["kv_heads"] * hd

    def r(rows, n, std=1.0):
        return torch.randn(rows, n, generator=g, device="cuda").mul_(std).to(dt)

    q, k, v = r(sum(ql), nq, 2.0), r(sum(kl), nk), r(sum(kl), nk)
    dout = r(sum(ql), nq) if c["train"] else None
    return q, k, v, dout


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = dict(case)
    if c["kind"] == "attn":
        q, k, v, dout = _attn_inputs(c, seed)
        ql, kl = _attn_lens(c)
        cu = _offsets(ql)
        state = {"case": c, "q": q, "k": k, "v": v, "dout": dout, "cu": cu,
                 "cu_k": _offsets(kl) if c["k_lens"] else cu, "max_q": max(ql), "max_k": max(kl)}
        leaves = (q, k, v)
    else:
        q, k, wq, wk, pos, dq, dk = _qk_inputs(c, seed)
        state = {"case": c, "q": q, "k": k, "wq": wq, "wk": wk, "pos": pos, "dq": dq, "dk": dk}
        leaves = (q, k, wq, wk)
    if c["train"]:
        for t in leaves:
            t.requires_grad_(True)
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _turns(c, pos):
    """cos and sin [..., N, 1, hd / 2] of every pair's angle: 64-bit angles, as far positions need."""
    ang = [pos[..., a:a + 1].double()
           * 10000.0 ** (torch.arange(0, d, 2, device=pos.device, dtype=torch.float64) / -d)
           for a, d in enumerate(_axes(c))]
    ang = torch.cat(ang, -1)[..., None, :]
    return ang.cos().float(), ang.sin().float()


def _pairs(c):
    """Channels of the first and of the second member of every pair."""
    first, second, at = [], [], 0
    for d in _axes(c):
        i = torch.arange(d // 2)
        first.append(at + (2 * i if c["interleaved"] else i))
        second.append(at + (2 * i + 1 if c["interleaved"] else i + d // 2))
        at += d
    return torch.cat(first).cuda(), torch.cat(second).cuda()


def _turn(x, cos, sin, first, second):
    a, b = x[..., first], x[..., second]
    y = torch.empty_like(x)
    y[..., first] = a * cos - b * sin
    y[..., second] = a * sin + b * cos
    return y


def _split(x, hd):
    return x.unflatten(-1, (-1, hd)).float()


def _plain_rope(s):
    c, hd = s["case"], s["case"]["head_dim"]
    (cos, sin), ch = _turns(c, s["pos"]), _pairs(c)
    y = _turn(_split(s["q"], hd), cos, sin, *ch).flatten(-2).to(s["q"].dtype)
    if not c["train"]:
        return y
    return y, _turn(_split(s["dq"], hd), cos, -sin, *ch).flatten(-2).to(y.dtype)


def _plain_norm_one(x, w, dy, hd, cos, sin, ch):
    dt, x, w = x.dtype, _split(x, hd), w.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    y = _turn(x * r * w, cos, sin, *ch).flatten(-2).to(dt)
    if dy is None:
        return y, None, None
    g = _turn(_split(dy, hd), cos, -sin, *ch)
    dw = (g * x * r).sum((0, 1, 2))
    g = g * w
    dx = r * g - x * (r ** 3 * (g * x).mean(-1, keepdim=True))
    return y, dx.flatten(-2).to(dt), dw


def _plain_norm(s):
    c, hd = s["case"], s["case"]["head_dim"]
    (cos, sin), ch = _turns(c, s["pos"]), _pairs(c)
    yq, dq, dwq = _plain_norm_one(s["q"], s["wq"], s["dq"], hd, cos, sin, ch)
    yk, dk, dwk = _plain_norm_one(s["k"], s["wk"], s["dk"], hd, cos, sin, ch)
    return (yq, yk, dq, dk, dwq, dwk) if c["train"] else (yq, yk)


def _pad(x, cu, most, heads):
    """Packed rows as [sequences, heads, most, hd]; rows behind a sequence's end are any rows."""
    at = (cu[:-1, None] + torch.arange(most, device=x.device)).clamp_max(x.shape[0] - 1)
    return x[at].float().unflatten(-1, (heads, -1)).transpose(1, 2)


def _unpad(x, cu, total, dt):
    """[sequences, heads, most, hd] back to packed rows."""
    row = torch.arange(total, device=x.device)
    seq = torch.bucketize(row, cu[1:].long(), right=True)
    return x.transpose(1, 2)[seq, row - cu[seq]].flatten(-2).to(dt)


def _plain_attn(s):
    c, cu, cu_k = s["case"], s["cu"].long(), s["cu_k"].long()
    q, k, v = s["q"].detach(), s["k"].detach(), s["v"].detach()
    hq, hk, hd = c["heads"], c["kv_heads"], c["head_dim"]
    Lq, Lk, dt = s["max_q"], s["max_k"], q.dtype
    scale = 1.0 / math.sqrt(hd)
    nq, nk = cu.diff()[:, None, None], cu_k.diff()[:, None, None]
    i = torch.arange(Lq, device=q.device)[:, None]
    j = torch.arange(Lk, device=q.device)[None, :]
    hide = (j >= nk) | (i >= nq)
    if c["causal"]:
        hide = hide | (j > i + (nk - nq))
    hide = hide[:, None, None]
    # the heads of a group as rows of one product with their keys
    qp = _pad(q, cu, Lq, hq).reshape(-1, hk, hq // hk * Lq, hd)
    kp, vp = _pad(k, cu_k, Lk, hk), _pad(v, cu_k, Lk, hk)

    def grouped(t):
        return t.view(t.shape[0], hk, hq // hk, Lq, Lk)

    p = torch.matmul(qp, kp.transpose(2, 3)).mul_(scale)
    grouped(p).masked_fill_(hide, -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
    out = torch.matmul(p, vp)
    heads = (-1, hq, Lq, hd)
    packed = _unpad(out.reshape(heads), cu, q.shape[0], dt)
    if not c["train"]:
        return packed
    do = _pad(s["dout"], cu, Lq, hq).reshape(qp.shape)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, vp.transpose(2, 3))
    ds.sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, kp).reshape(heads)
    dk = torch.matmul(ds.transpose(2, 3), qp)
    return (packed, _unpad(dq, cu, q.shape[0], dt), _unpad(dk, cu_k, k.shape[0], dt),
            _unpad(dv, cu_k, k.shape[0], dt))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _own(s):
    import megaslide_amd as ms
    c = s["case"]
    if c["kind"] == "attn":
        cu_k = s["cu_k"] if c["k_lens"] else None
        out = ms.packed_attention(s["q"], s["k"], s["v"], c["heads"], c["kv_heads"],
                                  cu_seqlens=s["cu"], cu_seqlens_k=cu_k, causal=c["causal"])
        if not c["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))
    if c["kind"] == "rope":
        y = ms.axial_rope(s["q"], s["pos"], c["heads"], axes=_axes(c),
                          interleaved=c["interleaved"])
        if not c["train"]:
            return y
        return y.detach(), torch.autograd.grad(y, s["q"], s["dq"])[0]
    yq, yk = ms.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["pos"], c["heads"],
                             c["kv_heads"], axes=_axes(c), eps=1e-6,
                             interleaved=c["interleaved"])
    if not c["train"]:
        return yq, yk
    leaves = (s["q"], s["k"], s["wq"], s["wk"])
    return (yq.detach(), yk.detach(), *torch.autograd.grad((yq, yk), leaves, (s["dq"], s["dk"])))


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        kind = state["case"]["kind"]
        if kind == "attn":
            return _plain_attn(state)
        return _plain_rope(state) if kind == "rope" else _plain_norm(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _visible(c):
    """(query, key) pairs that are not masked."""
    n = 0
    for a, b in zip(*_attn_lens(c)):
        if not c["causal"]:
            n += a * b
        elif a <= b:
            n += a * (b - a) + a * (a + 1) // 2
        else:
            n += b * (b + 1) // 2
    return n


def work(case):
    """Attention: 4 hd operations a visible pair and query head forward, 10 hd backward (five
    products); q, k, v (and dout) read, out (and three gradients) written.  Rotation and norm:
    x read, y written; in training dy read, dx written too."""
    c = case
    e = 2 if c["dtype"] == "bf16" else 4
    if c["kind"] == "attn":
        ql, kl = _attn_lens(c)
        rows = sum(ql) * c["heads"] + sum(kl) * c["kv_heads"]
        return {"bytes": e * c["head_dim"] * rows * (4 if c["train"] else 2),
                "flops": _visible(c) * c["heads"] * c["head_dim"] * (14 if c["train"] else 4)}
    n = c["B"] * c["T"] * c["H"] * c["W"]
    values = n * (c["heads"] + c["kv_heads"]) * c["head_dim"]
    per = (3 if c["kind"] == "rope" else 7) * (3 if c["train"] else 1)
    return {"bytes": e * values * (4 if c["train"] else 2) + 12 * n, "flops": per * values}


# ---------------------------------------------------------------------------
# float64 results
# ---------------------------------------------------------------------------

def _turn_exact(c, x, pos, sign):
    """x [B, N, heads, hd] as complex numbers, times exp(i sign angle)."""
    parts, at = [], 0
    for a, d in enumerate(_axes(c)):
        freq = torch.exp(torch.arange(d // 2, device=x.device).double()
                         * (-2.0 * math.log(10000.0) / d))
        ang = sign * pos[..., a].double()[..., None, None] * freq
        blk = x[..., at:at + d]
        blk = blk.unflatten(-1, (d // 2, 2)) if c["interleaved"] else \
            blk.unflatten(-1, (2, d // 2)).transpose(-1, -2)
        z = torch.view_as_complex(blk.contiguous()) * torch.polar(torch.ones_like(ang), ang)
        blk = torch.view_as_real(z)
        parts.append((blk if c["interleaved"] else blk.transpose(-1, -2)).flatten(-2))
        at += d
    return torch.cat(parts, -1)


def _qk_exact(c, seed):
    q, k, wq, wk, pos, dq, dk = _qk_inputs(c, seed)
    hd = c["head_dim"]
    pos = pos.expand(c["B"], *pos.shape[-2:])

    def one(x, w, dy):
        x = x.double().unflatten(-1, (-1, hd))
        dy = None if dy is None else _turn_exact(c, dy.double().unflatten(-1, (-1, hd)), pos, -1.0)
        if w is None:
            return (_turn_exact(c, x, pos, 1.0).flatten(-2),
                    None if dy is None else dy.flatten(-2), None)
        r = (x.pow(2).sum(-1, keepdim=True) / hd + 1e-6).pow(-0.5)
        n = x * r
        y = _turn_exact(c, n * w.double(), pos, 1.0).flatten(-2)
        if dy is None:
            return y, None, None
        g = dy * w.double()
        dx = r * (g - n * (g * n).mean(-1, keepdim=True))
        return y, dx.flatten(-2), (dy * n).sum((0, 1, 2))

    if c["kind"] == "rope":
        y, dx, _ = one(q, None, dq)
        return (y, dx) if c["train"] else y
    yq, gq, gwq = one(q, wq, dq)
    yk, gk, gwk = one(k, wk, dk)
    return (yq, yk, gq, gk, gwq, gwk) if c["train"] else (yq, yk)


def _attn_exact(c, seed):
    """One sequence and one head at a time, over the keys that each query sees."""
    q, k, v, dout = _attn_inputs(c, seed)
    hd, group = c["head_dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v))
    a0 = b0 = 0
    for a, b in zip(*_attn_lens(c)):
        rows, keys = slice(a0, a0 + a), slice(b0, b0 + b)
        a0, b0 = a0 + a, b0 + b
        if a == 0 or b == 0:
            continue
        seen = torch.ones(a, b, dtype=torch.bool, device=q.device)
        if c["causal"]:
            seen = seen.tril(b - a)
        empty = ~seen.any(1)
        for h in range(c["heads"]):
            ch = slice(h * hd, (h + 1) * hd)
            kv = slice(h // group * hd, (h // group + 1) * hd)
            kk, vv, qq = k[keys, kv].double(), v[keys, kv].double(), q[rows, ch].double()
            s = (qq @ kk.t() / math.sqrt(hd)).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, 1).masked_fill(empty[:, None], 0.0)
            o = p @ vv
            out[rows, ch] = o
            if dout is not None:
                g = dout[rows, ch].double()
                dv[keys, kv] += p.t() @ g
                dp = g @ vv.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(hd)
                dq[rows, ch] = ds @ kk
                dk[keys, kv] += ds.t() @ qq
    return (out, dq, dk, dv) if c["train"] else out


def exact(case, seed):
    with torch.no_grad():
        return _attn_exact(case, seed) if case["kind"] == "attn" else _qk_exact(case, seed)
