"""The dense operators as they are used together: norm and rotation, attention, a block around
them, training steps, packed clips, a step over a cache (GPU)."""

import math

import pytest
import torch

from dense_ref import attention, lens_to_cu, turn

pytestmark = pytest.mark.gpu

DEV = "cuda"


class Config:
    def __init__(self, dim, heads):
        self.hidden_size = dim
        self.num_heads = heads
        self.dsa_kernel_size = (3, 3, 3)
        self.offset_scale = 1.0
        self.dropout = 0.0
        self.mlp_hidden_size = 2 * dim
        self.use_text_conditioning = False


def dense_ref(m, p, x, positions, lens, axes):
    """DenseAttention3D in float64 with autograd, from parameters p."""
    def lin(t, n):
        return t @ p[n + ".weight"].t() + p[n + ".bias"]

    hd, out = m.head_dim, []
    qkv = [lin(x, n + "_proj") for n in "qkv"]
    heads = (m.num_heads, m.num_kv_heads)

    def prep(t, n, w):
        t = t.unflatten(-1, (n, hd))
        if w is not None:
            t = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        return turn(t, positions, axes, m.theta, False)

    q, k = prep(qkv[0], heads[0], p.get("q_norm")), prep(qkv[1], heads[1], p.get("k_norm"))
    v = qkv[2].unflatten(-1, (heads[1], hd))
    rep, at = heads[0] // heads[1], 0
    for n in lens:
        r = slice(at, at + n)
        at += n
        kk, vv = (t[r].repeat_interleave(rep, 1).transpose(0, 1) for t in (k, v))
        s = q[r].transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(hd)
        if m.causal:
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1),
                              -math.inf)
        out.append((torch.softmax(s, -1) @ vv).transpose(0, 1).flatten(1))
    return lin(torch.cat(out), "out_proj")


@pytest.mark.parametrize("kv,qk_norm,causal,packed", [
    (4, True, False, False), (2, True, True, True), (1, False, True, False), (4, False, False, True),
])
def test_module_against_float64(kv, qk_norm, causal, packed):
    """fp32 module, outputs and every gradient, at the fp32 parity tolerance 1e-4 of the largest
    element (the products of 128 to 2,000 terms and the chain of five fp32 stages stay well
    below)."""
    from megaslide_amd import DenseAttention3D, video_axes, video_positions
    torch.manual_seed(1)
    m = DenseAttention3D(128, 4, kv, qk_norm=qk_norm, causal=causal).to(DEV)
    with torch.no_grad():
        for n, t in m.named_parameters():
            if n.endswith("norm"):
                t.add_(0.2 * torch.randn_like(t))
    shapes = [(2, 5, 7), (1, 3, 4), (4, 6, 6)] if packed else [(3, 6, 7)]
    lens = [math.prod(s) for s in shapes]
    pos = torch.cat([video_positions(s, DEV) for s in shapes])
    x = torch.randn(sum(lens), 128, device=DEV)
    gy = torch.randn_like(x)
    xd = x.clone().requires_grad_(True)
    if packed:
        y = m(xd, positions=pos, cu_seqlens=lens_to_cu(lens, DEV))
    else:
        y = m(xd[None], shapes[0])[0]
    params = dict(m.named_parameters())
    grads = torch.autograd.grad(y, [xd, *params.values()], gy)
    p = {n: t.detach().double().requires_grad_(True) for n, t in params.items()}
    xr = x.double().requires_grad_(True)
    yr = dense_ref(m, p, xr, pos, lens, video_axes(32))
    want = torch.autograd.grad(yr, [xr, *p.values()], gy.double())
    for name, a, b in zip(["y", "x", *params], (y, *grads), (yr, *want)):
        scale = b.abs().max()
        if name == "k_proj.bias":  # without the norm a shift of every key: zero up to rounding
            scale = torch.maximum(scale, want[1 + list(p).index("k_proj.weight")].abs().max())
        assert float((a.double() - b).abs().max() / scale) < 1e-4, name


def test_block_trains_and_matches_its_deformable_form():
    """A DiTBlock with dense attention: forward, backward, checkpointing that keeps the
    attention; a block without the argument is the deformable one."""
    from megaslide_amd import (DeformableSlideAttention3D, DenseAttention3D, DiTBlock,
                               checkpoint_keep_core)
    torch.manual_seed(2)
    cfg = Config(256, 4)
    assert isinstance(DiTBlock(cfg).attn, DeformableSlideAttention3D)
    block = DiTBlock(cfg, DenseAttention3D(256, 4, 2)).to(DEV, torch.bfloat16)
    x = torch.randn(2, 3 * 8 * 9, 256, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    gy = torch.randn_like(x)
    params = [x, *block.parameters()]
    want = torch.autograd.grad(block(x, (3, 8, 9)), params, gy)
    assert all(torch.isfinite(g).all() for g in want)
    kept = torch.autograd.grad(checkpoint_keep_core(block, x, (3, 8, 9)), params, gy)
    assert all(torch.equal(a, b) for a, b in zip(want, kept))
    with torch.autocast("cuda", torch.bfloat16):
        y = DiTBlock(cfg, DenseAttention3D(256, 4)).to(DEV)(x.float(), (3, 8, 9))
    assert torch.isfinite(y).all()


def test_tokens_one_by_one_are_the_prompt():
    """A prompt at once, and the same tokens one by one over the cache they leave: the same rows
    within the roundings of the two calls."""
    from megaslide_amd import packed_attention, qk_norm_rope
    g = torch.Generator(device=DEV).manual_seed(3)
    heads, kv, hd, n, warm = 8, 2, 64, 1300, 1290
    q, k, v = (torch.randn(n, h * hd, generator=g, device=DEV).bfloat16()
               for h in (heads, kv, kv))
    w = torch.rand(hd, generator=g, device=DEV) + 0.5
    pos = torch.arange(n, device=DEV)[:, None]
    qr, kr = qk_norm_rope(q, k, w, w, pos, heads, kv)
    whole = packed_attention(qr, kr, v, heads, kv, causal=True)
    ref, err = attention(qr, kr, v, [n], [n], heads, kv, True)
    cu_q = lens_to_cu([1], DEV)
    for i in range(warm, n):
        qi, ki = qk_norm_rope(q[i:i + 1], k[i:i + 1], w, w, pos[i:i + 1], heads, kv)
        assert torch.equal(qi[0], qr[i]) and torch.equal(ki[0], kr[i])
        one = packed_attention(qi, kr, v, heads, kv, cu_q, lens_to_cu([i + 1], DEV), True)
        # each is within its bound of the exact row
        assert float(((one[0].double() - whole[i].double()).abs() - 2.02 * err[0][i]).max()) <= 0


def test_training_step_in_a_graph():
    """Norm, attention and their backward captured once, replayed on new inputs and offsets with
    eager work between the replays."""
    from megaslide_amd import packed_attention, qk_norm_rope
    g = torch.Generator(device=DEV).manual_seed(4)
    heads, kv, hd, n = 4, 2, 64, 500

    def make():
        return [torch.randn(n, h * hd, generator=g, device=DEV).bfloat16()
                for h in (heads, kv, kv, heads)]

    def step(q, k, v, dout, w, pos, cu):
        ins = [t.detach().requires_grad_(True) for t in (q, k, v, w)]
        qr, kr = qk_norm_rope(ins[0], ins[1], ins[3], ins[3], pos, heads, kv)
        out = packed_attention(qr, kr, ins[2], heads, kv, cu, causal=True)
        return [out.detach(), *torch.autograd.grad(out, ins, dout)]

    w = torch.rand(hd, generator=g, device=DEV) + 0.5
    pos = torch.arange(n, device=DEV, dtype=torch.int32)[:, None]
    static = [*make(), w, pos, lens_to_cu([100, 400], DEV)]
    step(*static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(*static)
    for lens in ([250, 250], [1, 499], [300, 0]):
        new = [*make(), w, pos, lens_to_cu(lens, DEV)]
        for s, t in zip(static, new):
            s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = step(*new)
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_module_refusals():
    from megaslide_amd import DenseAttention3D
    m = DenseAttention3D(64, 2).to(DEV)
    x = torch.zeros(1, 12, 64, device=DEV)
    with pytest.raises(ValueError, match="video_shape or positions"):
        m(x)
    with pytest.raises(ValueError, match="grid"):
        m(x, (2, 2, 2))
    with pytest.raises(RuntimeError, match="ROCm"):
        m(x.cpu(), (3, 2, 2))
    with pytest.raises(AssertionError):
        DenseAttention3D(64, 4, 3)
