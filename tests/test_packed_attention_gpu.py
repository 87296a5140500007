"""Attention over packed sequences against 64 bits (GPU)."""

import math

import pytest
import torch

from dense_ref import assert_within, attention, lens_to_cu

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dt=F32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)


def inputs(lq, lk, heads, kv, hd, dt, seed=0, std=1.5):
    g = gen(seed)
    q = randn(g, sum(lq), heads * hd, dt=dt, std=std)
    k, v = (randn(g, sum(lk), kv * hd, dt=dt) for _ in range(2))
    return q, k, v, randn(g, sum(lq), heads * hd, dt=dt)


def check(lq, lk, heads, kv, hd, dt, causal, seed=0, dlse=False, scale=None):
    from megaslide_amd import packed_attention
    q, k, v, dout = inputs(lq, lk, heads, kv, hd, dt, seed)
    gl = randn(gen(seed + 1), sum(lq), heads) if dlse else None
    for t in (q, k, v):
        t.requires_grad_(True)
    out, lse = packed_attention(q, k, v, heads, kv, lens_to_cu(lq, DEV), lens_to_cu(lk, DEV),
                                causal, scale, return_lse=True)
    if dlse:
        gl = torch.where(torch.isfinite(lse), gl, torch.zeros_like(gl))
        grads = torch.autograd.grad((out, lse), (q, k, v), (dout, gl))
    else:
        grads = torch.autograd.grad(out, (q, k, v), dout)
    with torch.no_grad():
        want, err = attention(q, k, v, lq, lk, heads, kv, causal, scale, dout, gl)
        for name, a, b, e in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads), want, err):
            assert_within(a, b, e, name)
        alone = packed_attention(q, k, v, heads, kv, lens_to_cu(lq, DEV), lens_to_cu(lk, DEV),
                                 causal, scale)
        assert torch.equal(alone, out)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hd", [1, 7, 8, 20, 32, 40, 64, 80, 96, 100, 128])
def test_head_sizes(dt, causal, hd):
    check([70, 1, 0, 133], [70, 1, 0, 133], 4, 2, hd, dt, causal)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 5), (6, 2), (8, 1), (7, 1), (40, 1), (3, 1)])
def test_groups(dt, causal, heads, kv):
    check([37, 90], [37, 90], heads, kv, 64, dt, causal)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [
    ([1], [1]),
    ([1, 1, 1], [1, 65, 300]),                 # single tokens over caches
    ([0, 0, 3], [5, 0, 0]),                    # sequences without queries, without keys
    ([64, 32, 128], [64, 32, 128]),            # whole tiles
    ([31, 33, 63, 65, 127, 129], [31, 33, 63, 65, 127, 129]),
    ([130, 40, 9], [20, 300, 1]),              # more queries than keys: rows that see nothing
    ([2, 5, 0, 17], [700, 64, 12, 1024]),      # a few new tokens over caches
    ([257], [513]),
])
def test_lengths(dt, causal, lq, lk):
    check(lq, lk, 4, 2, 64, dt, causal, dlse=True)


@pytest.mark.parametrize("S", [63, 64, 65, 130])
def test_many_sequences(S):
    lens = [(i * 7) % 23 for i in range(S)]
    check(lens, lens, 2, 1, 32, BF, True)
    check([1] * S, [(i * 37) % 190 for i in range(S)], 2, 1, 32, BF, True)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_long(dt, hd):
    """Keys split among workgroups, and many tiles."""
    check([1, 3], [5000, 2111], 8, 2, hd, dt, True)
    check([1500], [1500], 4, 4, hd, dt, True)
    check([300], [3001], 2, 1, hd, dt, False, scale=0.05)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("lq,lk,heads,kv,hd", [
    ([1] * 5, [1, 4000, 31, 33, 1025], 8, 2, 128),
    ([1] * 3, [0, 2500, 257], 4, 4, 64),             # a sequence without keys
    ([0, 2, 1], [700, 900, 1500], 6, 2, 96),         # as many tokens as sequences, not one each
    ([3, 0, 0], [2, 900, 600], 4, 1, 80),            # two tokens that see no key when causal
    ([1] * 70, [(i * 53) % 211 for i in range(70)], 32, 1, 32),  # more sequences than lanes
    ([1] * 2, [700, 1300], 33, 1, 64),               # a group beyond one block's rows
    ([1], [70001], 4, 1, 128),
])
def test_single_tokens(dt, lq, lk, heads, kv, hd):
    """One new token each over caches (and calls that only look like it)."""
    for causal in (True, False):
        check(lq, lk, heads, kv, hd, dt, causal)


def test_single_tokens_batched():
    """[B, 1, D] over [B, M, D], views with a batch stride, NaN behind every cache's end."""
    from megaslide_amd import packed_attention
    g = gen(11)
    B, M, heads, kv, hd = 6, 1003, 8, 2, 64
    q, k, v = (randn(g, B, n, h * hd, dt=BF) for n, h in ((1, heads), (M, kv), (M, kv)))
    want, err = attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), [1] * B, [M] * B,
                          heads, kv, True)
    out, lse = packed_attention(q, k, v, heads, kv, causal=True, return_lse=True)
    assert_within(out.flatten(0, 1), want[0], err[0], "out")
    assert_within(lse.flatten(0, 1), want[1], err[1], "lse")
    # caches with room for more keys than they hold, packed by offsets of their own rows
    room = 1500
    big = [torch.full((B * room, kv * hd), math.nan, dtype=BF, device=DEV) for _ in range(2)]
    for t, x in zip(big, (k, v)):
        t.view(B, room, -1)[:, :M] = x
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    for b in range(B):
        cu_k = (torch.tensor([0, M], dtype=torch.int32, device=DEV))
        rows = slice(b * room, (b + 1) * room)
        got = packed_attention(q[b], big[0][rows], big[1][rows], heads, kv,
                               torch.cat([one - 1, one]), cu_k, True)
        assert_within(got, want[0][b:b + 1], err[0][b:b + 1], "with room")


def test_seeded_shapes():
    """Random lengths, heads and sizes."""
    import random
    r = random.Random(3)
    for i in range(24):
        S = r.randint(1, 9)
        top = r.choice([3, 40, 200, 600])
        lk = [r.randint(0, top) for _ in range(S)]
        lq = lk if r.random() < 0.6 else [r.randint(0, top) for _ in range(S)]
        if sum(lq) == 0 or sum(lk) == 0:
            lq, lk = [1], [1]
        kv, grp = r.choice([1, 2, 3]), r.choice([1, 2, 3, 5])
        hd, dt, causal = r.choice([16, 24, 64, 72, 128]), r.choice([BF, F32]), r.random() < 0.6
        print(f"[attn] {i}: {lq} {lk} {kv * grp}/{kv}x{hd} {dt} {causal}", flush=True)
        check(lq, lk, kv * grp, kv, hd, dt, causal, seed=100 + i, dlse=r.random() < 0.3)


def test_gradient_against_differences():
    """The 64-bit form's own differences along a random direction."""
    from megaslide_amd import packed_attention
    lens, heads, kv, hd = [9, 30], 4, 2, 32
    q, k, v, dout = inputs(lens, lens, heads, kv, hd, F32)
    dirs = [randn(gen(9 + i), *t.shape) for i, t in enumerate((q, k, v))]
    for t in (q, k, v):
        t.requires_grad_(True)
    cu = lens_to_cu(lens, DEV)
    out = packed_attention(q, k, v, heads, kv, cu, causal=True)
    grads = torch.autograd.grad(out, (q, k, v), dout)

    def loss(t):
        x = [a.detach().double() + t * d.double() for a, d in zip((q, k, v), dirs)]
        tot, at = 0.0, 0
        for n in lens:
            r = slice(at, at + n)
            at += n
            for h in range(heads):
                c, ck = slice(h * hd, h * hd + hd), slice(h // 2 * hd, h // 2 * hd + hd)
                s = x[0][r, c] @ x[1][r, ck].t() / math.sqrt(hd)
                s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -math.inf)
                tot += float((torch.softmax(s, 1) @ x[2][r, ck] * dout[r, c].double()).sum())
        return tot

    diff = (loss(1e-5) - loss(-1e-5)) / 2e-5
    got = sum(float((a.double() * b.double()).sum()) for a, b in zip(grads, dirs))
    mag = sum(float((a.double() * b.double()).abs().sum()) for a, b in zip(grads, dirs))
    assert abs(got - diff) <= 1e-5 * mag


@pytest.mark.parametrize("dt", [BF, F32])
def test_batched_form_and_views(dt):
    """[B, N, D] without offsets, slices of a fused projection, unaligned rows, transposed
    storage: the same bits as packed contiguous rows."""
    from megaslide_amd import packed_attention
    g = gen(5)
    B, N, heads, kv, hd = 3, 77, 4, 2, 64
    fused = randn(g, B, N, (heads + 2 * kv) * hd, dt=dt)
    q, k, v = fused.split([heads * hd, kv * hd, kv * hd], -1)
    dout = randn(g, B, N, heads * hd, dt=dt)

    def call(q, k, v):
        ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = packed_attention(*ins, heads, kv, causal=True)
        return [out.detach(), *torch.autograd.grad(out, ins, dout)]

    want = call(*(t.contiguous() for t in (q, k, v)))
    with torch.no_grad():
        ref, err = attention(*(t.flatten(0, 1) for t in (q, k, v)), [N] * B, [N] * B, heads, kv,
                             True, dout=dout.flatten(0, 1))
    for a, b, e in zip(want, (ref[0], *ref[2:]), (err[0], *err[2:])):
        assert_within(a.flatten(0, 1), b, e, "batched")
    odd = randn(g, B * N * (kv * hd + 1) + 8, dt=dt)
    ko = odd[1:1 + B * N * (kv * hd + 1)].view(B, N, -1)[..., :kv * hd]
    ko.copy_(k)
    kt = k.transpose(0, 1).contiguous().transpose(0, 1)
    for kk in (k, ko, kt):
        got = call(q, kk, v)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    # one sequence without offsets
    one = packed_attention(q[0], k[0], v[0], heads, kv, causal=True)
    assert torch.equal(one, packed_attention(q[:1], k[:1], v[:1], heads, kv, causal=True)[0])


@pytest.mark.parametrize("dt", [BF, F32])
def test_rows_behind_the_last_sequence(dt):
    """Rows in no sequence, NaN there: out 0, lse -inf, gradients 0, the others untouched."""
    from megaslide_amd import packed_attention
    heads, kv, hd = 4, 2, 64
    lens = [50, 30]
    q, k, v, dout = inputs(lens, lens, heads, kv, hd, dt)
    pad = 200
    big = [torch.full((80 + pad, t.shape[1]), math.nan, dtype=dt, device=DEV)
           for t in (q, k, v, dout)]
    for b, t in zip(big, (q, k, v, dout)):
        b[:80] = t
    cu = lens_to_cu(lens, DEV)

    def call(q, k, v, dout):
        ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out, lse = packed_attention(*ins, heads, kv, cu, causal=True, return_lse=True)
        return [out.detach(), lse.detach(), *torch.autograd.grad(out, ins, dout)]

    want, got = call(q, k, v, dout), call(*big)
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a[:80], b)
        fill = -math.inf if i == 1 else 0.0
        assert torch.equal(a[80:], torch.full_like(a[80:], fill))


@pytest.mark.parametrize("S", [3, 63, 64, 100])
def test_rows_behind_many_sequences(S):
    """The same with more sequences than a wave has lanes, and as many tokens as sequences."""
    from megaslide_amd import packed_attention
    g = gen(S)
    for lq, lk in (([(i * 5) % 9 for i in range(S)], [(i * 5) % 9 for i in range(S)]),
                   ([1] * (S - 1) + [0], [(i * 31) % 77 for i in range(S)])):
        n, m = sum(lq), sum(lk)
        extra = 1 if lq[-1] == 0 and sum(lq) == S - 1 else 37
        q = randn(g, n + extra, 64, dt=BF)
        k, v = randn(g, m + 50, 32, dt=BF), randn(g, m + 50, 32, dt=BF)
        q[n:], k[m:], v[m:] = math.nan, math.nan, math.nan
        ins = [t.requires_grad_(True) for t in (q, k, v)]
        out = packed_attention(q, k, v, 2, 1, lens_to_cu(lq, DEV), lens_to_cu(lk, DEV), True)
        dout = randn(g, n + extra, 64, dt=BF)
        grads = torch.autograd.grad(out, ins, dout)
        with torch.no_grad():
            want, err = attention(q[:n], k[:m], v[:m], lq, lk, 2, 1, True, dout=dout[:n])
            for a, b, e, r in zip((out, *grads), (want[0], *want[2:]), (err[0], *err[2:]),
                                  (n, n, m, m)):
                assert_within(a[:r], b, e, "rows")
                assert not a[r:].any()


def test_strides_and_offsets_beyond_32_bits():
    """Keys and values whose rows lie further apart than a tile's 32-bit offsets reach, and whose
    last rows lie beyond 2^32 bytes and elements of the first: the bits of contiguous ones."""
    from megaslide_amd import packed_attention
    g = gen(21)
    heads, kv, hd = 4, 2, 64
    for n, stride in ((2100, 1 << 21), (9, (1 << 22) + 8)):
        print(f"[attn] {n} rows {stride} apart", flush=True)
        k, v = randn(g, n, kv * hd, dt=BF), randn(g, n, kv * hd, dt=BF)
        q = randn(g, n, heads * hd, dt=BF)
        big = torch.empty(n * stride, dtype=BF, device=DEV).view(n, stride)
        kb, vb = big[:, :kv * hd], big[:, 512:512 + kv * hd]
        kb.copy_(k)
        vb.copy_(v)

        def call(q, k, v):
            ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
            out = packed_attention(*ins, heads, kv, causal=True)
            return [out.detach(), *torch.autograd.grad(out, ins, q)]

        assert all(torch.equal(a, b) for a, b in zip(call(q, kb, vb), call(q, k, v)))
        cu = lens_to_cu([1], DEV), lens_to_cu([n], DEV)  # one token over the cache
        assert torch.equal(packed_attention(q[:1], kb, vb, heads, kv, *cu),
                           packed_attention(q[:1], k, v, heads, kv, *cu))
        del big, kb, vb


def test_saved_tensors():
    """A backward that is run twice, and one after its inputs were written to (an error)."""
    from megaslide_amd import packed_attention, qk_norm_rope
    q, k, v, dout = inputs([40], [40], 2, 2, 32, BF)
    for t in (q, k, v):
        t.requires_grad_(True)
    out = packed_attention(q, k, v, 2, causal=True)
    a = torch.autograd.grad(out, (q, k, v), dout, retain_graph=True)
    b = torch.autograd.grad(out, (q, k, v), dout)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    pos = torch.arange(40, device=DEV)[:, None]
    w = torch.ones(32, device=DEV)
    for change in (lambda: v.detach().mul_(2), lambda: pos.add_(1), lambda: w.add_(1)):
        qr, kr = qk_norm_rope(q, k, w, w, pos, 2)
        out = packed_attention(qr, kr, v, 2, causal=True)
        change()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, (q, k, v), dout)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("hd", [32, 128])
def test_nonfinite_values_stay_where_they_are_seen(dt, hd):
    """NaN and infinities in later keys and values, in other sequences and in other rows'
    gradients: what does not see them keeps its bits."""
    from megaslide_amd import packed_attention
    heads, kv = 4, 2
    lens = [75, 140]
    q, k, v, dout = inputs(lens, lens, heads, kv, hd, dt)
    cu = lens_to_cu(lens, DEV)

    def call(q, k, v, dout):
        ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = packed_attention(*ins, heads, kv, cu, causal=True)
        return [out.detach(), *torch.autograd.grad(out, ins, dout)]

    want = call(q, k, v, dout)
    row = 75 + 99  # in the second sequence, inside a tile
    for which, val in ((0, math.nan), (1, math.nan), (2, math.nan), (2, math.inf), (2, -math.inf),
                       (1, math.inf), (3, math.nan), (3, math.inf), (0, math.inf)):
        ins = [t.clone() for t in (q, k, v, dout)]
        ins[which][row] = val
        got = call(*ins)
        # rows of the first sequence, and rows before the bad one
        early = torch.arange(215, device=DEV) < row
        first = torch.arange(215, device=DEV) < 75
        assert torch.equal(got[0][early], want[0][early]), (which, val)
        assert torch.equal(got[1][early], want[1][early]), (which, val)
        assert torch.equal(got[2][first], want[2][first]), (which, val)
        assert torch.equal(got[3][first], want[3][first]), (which, val)
        # keys after the bad query are not seen by it: their gradients stay
        if which in (0, 3):
            late = torch.arange(215, device=DEV) > row
            assert torch.equal(got[2][late], want[2][late]), (which, val)
            assert torch.equal(got[3][late], want[3][late]), (which, val)
        # and it is not lost where it is seen
        if which in (0, 1):
            assert not torch.isfinite(got[0][row]).any()
        if which == 2:
            assert torch.isnan(got[0][row:]).all() if val != val else \
                torch.equal(got[0][row:], torch.full_like(got[0][row:], val))
        if which == 3:
            assert not torch.isfinite(got[3][75:row + 1]).any()


def test_repeats_bit_for_bit_and_across_batch():
    """The same bits on every run, and a sequence's results do not depend on its neighbours."""
    from megaslide_amd import packed_attention
    lens, heads, kv, hd = [300, 41, 517], 4, 1, 128
    q, k, v, dout = inputs(lens, lens, heads, kv, hd, BF)

    def call(q, k, v, dout, lens):
        ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = packed_attention(*ins, heads, kv, lens_to_cu(lens, DEV), causal=True)
        return [out.detach(), *torch.autograd.grad(out, ins, dout)]

    want = call(q, k, v, dout, lens)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(call(q, k, v, dout, lens), want))


def test_streams_devices_and_graph():
    """On a side stream; captured (forward and backward) and replayed with other contents and
    other lengths, which the kernels read on the device."""
    from megaslide_amd import packed_attention
    heads, kv, hd = 4, 2, 64
    total, most = 400, [250, 150]
    q, k, v, dout = inputs(most, most, heads, kv, hd, BF)
    cu = lens_to_cu(most, DEV)

    def step(q, k, v, dout, cu):
        ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = packed_attention(*ins, heads, kv, cu, causal=True)
        return [out.detach(), *torch.autograd.grad(out, ins, dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(q, k, v, dout, cu)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, step(q, k, v, dout, cu)))

    static = [t.clone() for t in (q, k, v, dout, cu)]
    graph, decode = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    cu1 = lens_to_cu([1, 1], DEV)
    with torch.cuda.graph(graph):
        res = step(*static)
    with torch.cuda.graph(decode):
        tok = packed_attention(static[0][:2], static[1], static[2], heads, kv, cu1, static[4],
                               causal=True)
    for seed, lens in ((31, [250, 150]), (32, [1, 399]), (33, [0, 210])):
        new = [*inputs([total], [total], heads, kv, hd, BF, seed), lens_to_cu(lens, DEV)]
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        decode.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, step(*new)))
        assert torch.equal(tok, packed_attention(new[0][:2], new[1], new[2], heads, kv, cu1,
                                                 new[4], causal=True))


@pytest.mark.parametrize("dt", [BF, F32])
def test_single_tokens_in_graphs_and_on_two_streams(dt):
    """Tokens over caches long enough to be joined from chunks: two captured graphs replayed in
    turn with other lengths, and two calls at a time on two streams."""
    from megaslide_amd import packed_attention
    heads, kv, hd, total = 8, 2, 64, 3000
    q, k, v, _ = inputs([1] * 3, [total], heads, kv, hd, dt)
    cu = lens_to_cu([1, 1, 1], DEV)

    def step(q, k, v, cu_k):
        return packed_attention(q, k, v, heads, kv, cu, cu_k, True, return_lse=True)

    static = [[t.clone() for t in (q, k, v, lens_to_cu([1000, 1000, 1000], DEV))]
              for _ in range(2)]
    graphs, res = [], []
    for s in static:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            res.append(step(*s))
    for seed, lens in ((41, [1000, 1000, 1000]), (42, [1, 2998, 1]), (43, [0, 17, 1500])):
        new = []
        for i, s in enumerate(static):
            qi, ki, vi, _ = inputs([1] * 3, [total], heads, kv, hd, dt, seed + 10 * i)
            new.append([qi, ki, vi, lens_to_cu(lens, DEV)])
            for x, y in zip(s, new[-1]):
                x.copy_(y)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for r, n in zip(res, new):
            assert all(torch.equal(x, y) for x, y in zip(r, step(*n)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st, n in zip(streams, new):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append([step(*n) for _ in range(3)])
    torch.cuda.synchronize()
    for calls, n in zip(got, new):
        want = step(*n)
        assert all(torch.equal(x, y) for c in calls for x, y in zip(c, want))


def test_offsets_out_of_order_stay_inside():
    """Offsets that break the documented order are held to the tensors' rows (their results are
    not defined): the calls end, and what follows on the same tensors is right."""
    from megaslide_amd import packed_attention
    heads, kv, hd = 2, 1, 32
    g = gen(3)
    for cu in ([0, 90, 40, 60], [0, -5, 1000, 60], [7, 20, 30, 60], [0, 0, 0, 0]):
        c = torch.tensor(cu, dtype=torch.int32, device=DEV)
        q, k, v = randn(g, 60, 64, dt=BF), randn(g, 60, 32, dt=BF), randn(g, 60, 32, dt=BF)
        for t in (q, k, v):
            t.requires_grad_(True)
        print(f"[attn] offsets {cu}", flush=True)
        out = packed_attention(q, k, v, heads, kv, c, causal=True)
        torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
        torch.cuda.synchronize()
    check([20, 40], [20, 40], heads, kv, hd, BF, True)


def test_empty_calls():
    from megaslide_amd import packed_attention
    q = torch.empty(0, 128, device=DEV, requires_grad=True)
    cu = torch.zeros(3, dtype=torch.int32, device=DEV)
    k = torch.randn(5, 64, device=DEV, requires_grad=True)
    out = packed_attention(q, k, k, 4, 2, cu, cu)
    dq, dk = torch.autograd.grad(out, (q, k), torch.empty_like(out))
    assert out.shape == (0, 128) and dq.shape == (0, 128)
    assert torch.equal(dk, torch.zeros_like(dk))
    q = torch.randn(5, 128, device=DEV, requires_grad=True)
    k = torch.empty(0, 64, device=DEV, requires_grad=True)
    out, lse = packed_attention(q, k, k, 4, 2, cu, cu, return_lse=True)
    (dq,) = torch.autograd.grad(out, q, torch.ones_like(out))
    assert not out.any() and not dq.any() and (lse == -math.inf).all()
    b = torch.empty(0, 7, 128, device=DEV)
    assert packed_attention(b, b, b, 4).shape == b.shape


def test_saved_tensors_of_another_layout():
    """Hooks on saved tensors hand back contiguous copies of the views that were saved."""
    from megaslide_amd import packed_attention
    g = gen(9)
    qkv = randn(g, 150, 8 * 64, dt=BF).requires_grad_(True)
    cu = lens_to_cu([70, 80], DEV)

    def f():
        q, k, v = qkv.split([256, 128, 128], -1)
        return packed_attention(q, k, v, 4, 2, cu, causal=True)

    dout = randn(g, 150, 256, dt=BF)
    (want,) = torch.autograd.grad(f(), qkv, dout)
    with torch.autograd.graph.save_on_cpu():
        out = f()
    (got,) = torch.autograd.grad(out, qkv, dout)
    assert torch.equal(got, want)


def test_checkpoint_keeps_the_attention():
    """The selective policy that keeps the deformable core's outputs keeps this one's too."""
    from torch.utils.checkpoint import checkpoint

    import megaslide_amd as ms
    q, k, v, dout = inputs([200], [200], 4, 2, 64, BF)
    for t in (q, k, v):
        t.requires_grad_(True)

    def f(q, k, v):
        return ms.packed_attention(q * 1.0, k, v, 4, 2, causal=True) * 1.0

    want = torch.autograd.grad(f(q, k, v), (q, k, v), dout)
    out = checkpoint(f, q, k, v, use_reentrant=False, context_fn=ms.keep_core_context)
    from megaslide_amd import dense_ops
    calls, real = [], dense_ops._AttnCall.forward
    dense_ops._AttnCall.forward = lambda self, *a, **kw: calls.append(1) or real(self, *a, **kw)
    try:
        got = torch.autograd.grad(out, (q, k, v), dout)
    finally:
        dense_ops._AttnCall.forward = real
    assert not calls
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    from megaslide_amd import packed_attention
    q, k = torch.zeros(10, 128, device=DEV), torch.zeros(10, 64, device=DEV)
    cu = lens_to_cu([10], DEV)
    with pytest.raises(ValueError, match="multiple"):
        packed_attention(q, q, q, 4, 3)
    with pytest.raises(ValueError, match="channels"):
        packed_attention(q, k, k, 4, 4)
    with pytest.raises(ValueError, match="differ"):
        packed_attention(q, k, k[:9], 4, 2)
    with pytest.raises(TypeError, match="k is"):
        packed_attention(q, k.bfloat16(), k, 4, 2)
    with pytest.raises(TypeError, match="dtype"):
        packed_attention(q.half(), k.half(), k.half(), 4, 2)
    with pytest.raises(ValueError, match="int32"):
        packed_attention(q, k, k, 4, 2, cu.long())
    with pytest.raises(ValueError, match="sequences"):
        packed_attention(q, k, k, 4, 2, cu, lens_to_cu([5, 5], DEV))
    with pytest.raises(ValueError, match="cu_seqlens_k"):
        packed_attention(q, k, k, 4, 2, cu_seqlens_k=cu)
    with pytest.raises(ValueError, match="rows"):
        packed_attention(q, k[:5], k[:5], 4, 2, cu)
    with pytest.raises(RuntimeError, match="scale"):
        packed_attention(q, k, k, 4, 2, cu, scale=-1.0)
    with pytest.raises(RuntimeError, match="head_dim"):
        packed_attention(torch.zeros(4, 256, device=DEV), *[torch.zeros(4, 256, device=DEV)] * 2, 1)
    with pytest.raises(RuntimeError, match="ROCm"):
        packed_attention(q.cpu(), k, k, 4, 2)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad|backward"):
        x = q.clone().requires_grad_(True)
        (g1,) = torch.autograd.grad(packed_attention(x, k, k, 4, 2).sum(), x, create_graph=True)
        torch.autograd.grad(g1.sum(), x)
