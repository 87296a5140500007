"""Rotary positions with several axes and the norm of queries and keys, against 64 bits (GPU)."""

import math

import pytest
import torch

from dense_ref import HALF, assert_within, norm_rope, turn

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def randn(g, *shape, dt=F32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("B,T,H,W,heads,hd,axes", [
    (1, 1, 1, 1, 1, 2, (2, 0, 0)),          # one token, one pair
    (1, 2, 3, 5, 4, 64, None),              # the usual split
    (2, 3, 4, 5, 3, 96, (32, 32, 32)),
    (1, 2, 2, 3, 2, 20, (4, 8, 6)),         # no multiple of 8, two channels pass through
    (1, 3, 2, 2, 5, 33, (12, 10, 10)),      # an odd head size
    (1, 4, 3, 3, 2, 128, (44, 42, 42)),
    (3, 1, 5, 7, 1, 256, None),
    (1, 2, 2, 2, 2, 72, (0, 36, 36)),       # an axis without channels
    (1, 8, 33, 37, 3, 40, None),            # more tokens than a workgroup's step
])
def test_rope_grid(dt, inter, B, T, H, W, heads, hd, axes):
    from megaslide_amd import axial_rope, video_axes, video_positions
    g = gen(1)
    x = randn(g, B, T * H * W, heads * hd, dt=dt).requires_grad_(True)
    dy = randn(g, B, T * H * W, heads * hd, dt=dt)
    ax = video_axes(hd) if axes is None else axes
    pos = video_positions((T, H, W), DEV)
    want, err = norm_rope(x.detach(), None, pos, heads, ax, 10000.0, 0.0, inter, dy, norm=False)
    y = axial_rope(x, (T, H, W), heads, axes=axes, interleaved=inter)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert_within(y, want[0], err[0], "y")
    assert_within(dx, want[1], err[1], "dx")
    # positions as a tensor give the same bits, and so does a call that saves nothing
    with torch.no_grad():
        assert torch.equal(axial_rope(x, pos, heads, axes=axes, interleaved=inter), y)


@pytest.mark.parametrize("pdt", [torch.int32, torch.int64, F32, torch.float64])
def test_rope_far_positions(pdt):
    """Angles of positions near 10^6 (2^24 for fp32 positions) keep their accuracy."""
    from megaslide_amd import axial_rope
    g = gen(2)
    x = randn(g, 2, 50, 4 * 64)
    pos = torch.randint(900000, 1000000, (2, 50, 1), generator=g, device=DEV).to(pdt)
    if pos.is_floating_point():
        pos = pos + 0.25
    want, err = norm_rope(x, None, pos, 4, (64,), 500000.0, 0.0, True, norm=False)
    y = axial_rope(x, pos, 4, theta=500000.0, interleaved=True)
    assert_within(y, want[0], err[0], "y")


def test_rope_negative_positions_undo():
    from megaslide_amd import axial_rope
    g = gen(3)
    x = randn(g, 60, 2 * 64)
    pos = torch.randint(-500, 500, (60, 2), generator=g, device=DEV)
    y = axial_rope(axial_rope(x, pos, 2, axes=(32, 32)), -pos, 2, axes=(32, 32))
    # two turns, 11 steps each, of magnitudes that a turn grows at most by sqrt 2
    assert float((y - x).abs().max()) <= 2 * 11 * 2.0 ** -24 * 2 * 2 * float(x.abs().max())


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("wdt", ["same", "fp32", "none"])
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("N,heads,kv,hd,axes", [
    (1, 1, 1, 2, (2,)),
    (1, 32, 8, 128, (128,)),
    (70, 4, 2, 64, (24, 20, 20)),
    (33, 6, 1, 96, (30, 30, 30)),
    (17, 3, 3, 20, (6, 6, 6)),
    (9, 5, 5, 33, (10, 10, 10)),
    (2100, 2, 1, 80, (28, 26, 26)),
])
def test_norm_rope(dt, wdt, inter, N, heads, kv, hd, axes):
    from megaslide_amd import qk_norm_rope
    g = gen(4)
    w0 = F32 if wdt == "fp32" else dt
    q, k = randn(g, 2, N, heads * hd, dt=dt, std=3), randn(g, 2, N, kv * hd, dt=dt, std=0.2)
    wq, wk = (1 + randn(g, hd, std=0.3)).to(w0), (1 + randn(g, hd, std=0.3)).to(w0)
    if wdt == "none":
        wq = wk = None
    pos = torch.randint(0, 300, (N, len(axes)), generator=g, device=DEV, dtype=torch.int32)
    dq, dk = randn(g, 2, N, heads * hd, dt=dt), randn(g, 2, N, kv * hd, dt=dt)
    leaves = [t for t in (q, k, wq, wk) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    yq, yk = qk_norm_rope(q, k, wq, wk, pos, heads, kv, axes=axes, interleaved=inter)
    grads = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    with torch.no_grad():
        for x, w, dy, h, y, dx, dw, name in (
                (q, wq, dq, heads, yq, grads[0], grads[2] if wq is not None else None, "q"),
                (k, wk, dk, kv, yk, grads[1], grads[3] if wk is not None else None, "k")):
            want, err = norm_rope(x, w, pos, h, axes, 10000.0, 1e-6, inter, dy)
            assert_within(y, want[0], err[0], name)
            assert_within(dx, want[1], err[1], "d" + name)
            if dw is not None:
                e = err[2] + HALF[dw.dtype] * want[2].abs()
                assert_within(dw, want[2], e, f"d{name}_weight")
        # results repeat bit for bit
    yq2, yk2 = qk_norm_rope(q, k, wq, wk, pos, heads, kv, axes=axes, interleaved=inter)
    again = torch.autograd.grad((yq2, yk2), leaves, (dq, dk))
    assert torch.equal(yq, yq2) and torch.equal(yk, yk2)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_norm_rope_gradient_against_differences():
    """The 64-bit form's own differences along a random direction."""
    from megaslide_amd import qk_norm_rope
    g = gen(5)
    N, heads, kv, hd, axes = 12, 3, 1, 64, (24, 20, 20)
    ins = [randn(g, N, heads * hd), randn(g, N, kv * hd), 1 + randn(g, hd, std=0.2),
           1 + randn(g, hd, std=0.2)]
    pos = torch.randint(0, 50, (N, 3), generator=g, device=DEV, dtype=torch.int32)
    dys = [randn(g, N, heads * hd), randn(g, N, kv * hd)]
    dirs = [randn(g, *t.shape) for t in ins]
    for t in ins:
        t.requires_grad_(True)
    ys = qk_norm_rope(*ins, pos, heads, kv, axes=axes)
    grads = torch.autograd.grad(ys, ins, dys)

    def loss(t):
        x = [i.detach().double() + t * d.double() for i, d in zip(ins, dirs)]
        tot = 0.0
        for X, Wt, n, dy in ((x[0], x[2], heads, dys[0]), (x[1], x[3], kv, dys[1])):
            X = X.unflatten(-1, (n, hd))
            r = (X.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
            Y = turn(X * r * Wt, pos, axes, 10000.0, False)
            tot += float((Y.flatten(-2) * dy.double()).sum())
        return tot

    step = 1e-5  # second-order term 1e-10 of the third derivative, 64-bit noise 1e-11
    diff = (loss(step) - loss(-step)) / (2 * step)
    got = sum(float((a.double() * b.double()).sum()) for a, b in zip(grads, dirs))
    mag = sum(float((a.double() * b.double()).abs().sum()) for a, b in zip(grads, dirs))
    assert abs(got - diff) <= 1e-5 * mag


@pytest.mark.parametrize("dt", [BF, F32])
def test_views_and_alignment(dt):
    """Slices of a fused projection, rows that are not 16-byte aligned, transposed storage, a
    batch stride that is no multiple of the token stride: the same bits as contiguous copies."""
    from megaslide_amd import axial_rope, qk_norm_rope
    g = gen(6)
    B, N, heads, kv, hd = 2, 30, 4, 2, 64
    fused = randn(g, B, N, (heads + 2 * kv) * hd, dt=dt)
    q, k = fused[..., :heads * hd], fused[..., heads * hd:(heads + kv) * hd]
    w = 1 + randn(g, hd, std=0.2)
    pos = torch.randint(0, 90, (B, N, 3), generator=g, device=DEV)

    def call(q, k):
        qd, kd = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        ys = qk_norm_rope(qd, kd, w, None, pos, heads, kv)
        return [*ys, *torch.autograd.grad(ys, (qd, kd), (q.detach(), k.detach()))]

    want = call(q.contiguous(), k.contiguous())
    odd = randn(g, B * N * (heads * hd + 3) + 8, dt=dt)
    qo = odd[1:1 + B * N * (heads * hd + 3)].view(B, N, -1)[..., :heads * hd]
    qo.copy_(q)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    qc = q.transpose(1, 2).contiguous().transpose(1, 2)
    for qv in (q, qo, qt, qc):
        assert all(torch.equal(a, b) for a, b in zip(call(qv, k), want))
    one = axial_rope(q[:, :1], pos[:, :1], heads)
    assert torch.equal(one, axial_rope(q[:, :1].contiguous(), pos[:, :1], heads))
    # an expanded tensor, and one query row for all heads' worth of tokens
    ex = q[:1, :1].expand(B, N, -1)
    assert torch.equal(axial_rope(ex, pos, heads), axial_rope(ex.contiguous(), pos, heads))


def test_empty_and_nonfinite():
    from megaslide_amd import axial_rope, qk_norm_rope
    x = torch.empty(0, 128, device=DEV, requires_grad=True)
    y = axial_rope(x, torch.empty(0, 3, device=DEV), 2)
    assert y.shape == x.shape
    w = torch.ones(64, device=DEV, requires_grad=True)
    yq, yk = qk_norm_rope(x, x, w, None, torch.empty(0, 3, device=DEV), 2)
    (dw,) = torch.autograd.grad((yq, yk), w, (torch.empty_like(yq),) * 2)
    assert torch.equal(dw, torch.zeros_like(dw))
    # a NaN or infinity stays in its own head of its own token
    g = gen(7)
    q = randn(g, 40, 4 * 64, dt=BF)
    bad = q.clone()
    bad[3, 64 + 5] = math.nan
    bad[7, 130] = math.inf
    pos = torch.arange(40, device=DEV)[:, None]
    good, _ = qk_norm_rope(q, q, None, None, pos, 4)
    got, _ = qk_norm_rope(bad, q, None, None, pos, 4)
    hit = torch.zeros(40, 4, dtype=torch.bool, device=DEV)
    hit[3, 1] = hit[7, 2] = True
    diff = (good != got).view(40, 4, 64).any(-1)
    assert torch.equal(diff, hit)
    # channels that no axis turns pass through, infinities too
    x = randn(g, 40, 2 * 32)
    x[5, 30] = math.inf
    y = axial_rope(x, pos, 2, axes=(16,))
    assert torch.equal(y.view(40, 2, 32)[..., 16:], x.view(40, 2, 32)[..., 16:])
    # a row of zeros: the norm's eps alone
    z = torch.zeros(3, 64, device=DEV, requires_grad=True)
    yz, _ = qk_norm_rope(z, z.detach(), None, None, pos[:3], 1, eps=1e-6)
    (dz,) = torch.autograd.grad(yz, z, torch.ones_like(yz))
    assert torch.equal(yz, torch.zeros_like(yz)) and torch.isfinite(dz).all()


@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("heads,kv,hd", [(16, 16, 64), (20, 4, 96), (9, 9, 128), (33, 33, 32)])
def test_results_past_the_caches(heads, kv, hd, inter):
    """Results of more than 128 MB are stored another way: the bits of calls on their parts."""
    from megaslide_amd import qk_norm_rope
    g = gen(12)
    n = (135 << 20) // (2 * (heads + kv) * hd)
    q, k, dq, dk = (randn(g, n, h * hd, dt=BF) for h in (heads, kv, heads, kv))
    w = [randn(g, hd) for _ in range(2)]
    pos = torch.randint(0, 500, (n, 3), generator=g, device=DEV, dtype=torch.int32)

    def f(rows):
        ins = [t[rows].requires_grad_(True) for t in (q, k)]
        y = qk_norm_rope(*ins, *w, pos[rows], heads, kv, interleaved=inter)
        return [t.detach() for t in y] + list(
            torch.autograd.grad(y, ins, (dq[rows], dk[rows])))

    whole = f(slice(None))
    for rows in (slice(0, n // 2), slice(n // 2, n)):
        for a, b in zip(whole, f(rows)):
            assert torch.equal(a[rows], b)


def test_saved_tensors_of_another_layout():
    """Hooks on saved tensors hand back contiguous copies of the views that were saved."""
    from megaslide_amd import qk_norm_rope
    g = gen(10)
    qkv = randn(g, 60, 6 * 64, dt=BF).requires_grad_(True)
    w = [randn(g, 64).requires_grad_(True) for _ in range(2)]
    dq, dk = randn(g, 60, 128, dt=BF), randn(g, 60, 128, dt=BF)

    def f():
        q, k, _ = qkv.split(128, -1)
        return qk_norm_rope(q, k, *w, (3, 4, 5), 2)

    want = torch.autograd.grad(f(), (qkv, *w), (dq, dk))
    with torch.autograd.graph.save_on_cpu():
        out = f()
    got = torch.autograd.grad(out, (qkv, *w), (dq, dk))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    empty = qkv[:0, :128]
    assert qk_norm_rope(empty, empty, None, None, (0, 4, 5), 2)[0].shape == (0, 128)


def test_streams_and_graph():
    """On a side stream, and captured with its backward and replayed on new contents."""
    from megaslide_amd import qk_norm_rope
    g = gen(8)
    B, T, H, W, heads, hd = 1, 3, 8, 8, 4, 64
    q, k = (randn(g, B, T * H * W, heads * hd, dt=BF) for _ in range(2))
    w = [1 + randn(g, hd, std=0.1) for _ in range(2)]
    dq, dk = (randn(g, B, T * H * W, heads * hd, dt=BF) for _ in range(2))

    def step(q, k, wq, wk, dq, dk):
        ins = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
        ys = qk_norm_rope(*ins, (T, H, W), heads)
        return [t.detach() for t in ys] + list(torch.autograd.grad(ys, ins, (dq, dk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(q, k, *w, dq, dk)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, step(q, k, *w, dq, dk)))

    static = [t.clone() for t in (q, k, *w, dq, dk)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(*static)
    for seed in (20, 21, 22):
        gg = gen(seed)
        new = [randn(gg, *t.shape, dt=t.dtype) for t in static]
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want = step(*new)
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_refusals():
    from megaslide_amd import axial_rope, qk_norm_rope
    x = torch.zeros(2, 12, 128, device=DEV)
    pos = torch.zeros(12, 3, device=DEV, dtype=torch.int32)
    with pytest.raises(ValueError, match="heads"):
        axial_rope(x, pos, 3)
    with pytest.raises(ValueError, match="even"):
        axial_rope(x, pos, 2, axes=(3, 3, 4))
    with pytest.raises(ValueError, match="even"):
        axial_rope(x, pos, 2, axes=(32, 32, 32))
    with pytest.raises(ValueError, match="axes"):
        axial_rope(x, pos, 2, axes=(32, 32))
    with pytest.raises(ValueError, match="positions"):
        axial_rope(x, pos[:11], 2)
    with pytest.raises(TypeError, match="positions"):
        axial_rope(x, pos.to(torch.int16), 2)
    with pytest.raises(ValueError, match="grid"):
        axial_rope(x, (2, 2, 2), 2)
    with pytest.raises(TypeError, match="dtype"):
        axial_rope(x.half(), pos, 2)
    with pytest.raises(RuntimeError, match="theta"):
        axial_rope(x, pos, 2, theta=0.0)
    with pytest.raises(ValueError, match="k must be"):
        qk_norm_rope(x, x, None, None, pos, 2, 1)
    with pytest.raises(TypeError, match="k is"):
        qk_norm_rope(x, x.bfloat16(), None, None, pos, 2)
    with pytest.raises(ValueError, match="q_weight"):
        qk_norm_rope(x, x, torch.ones(32, device=DEV), None, pos, 2)
    with pytest.raises(RuntimeError, match="eps"):
        qk_norm_rope(x, x, None, None, pos, 2, eps=-1.0)
    with pytest.raises(RuntimeError, match="ROCm"):
        axial_rope(x.cpu(), pos, 2)
