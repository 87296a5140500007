"""Operators of dense attention layers over the HIP kernels.

``axial_rope``        rotary positions with several axes (time, height, width)
``qk_norm_rope``      RMS norm of each head of queries and keys and that rotation, in one pass
``packed_attention``  attention over sequences of different lengths packed into one call, with
                      grouped heads, causal or full, as the custom operators
                      megaslide::packed_attention (+ _bwd)

They serve the layers that attend to everything (the reference's dense baseline,
infinity/video/baselines.py, and its decoder layers) beside the deformable slide attention, and
take tensors as it does: [B, N, heads * head_dim], token-major, or packed rows
[N, heads * head_dim].  They run only on ROCm device tensors; there is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib

Tensor = torch.Tensor
Positions = Union[Tensor, Sequence[int]]


def video_axes(head_dim: int) -> Tuple[int, int, int]:
    """Channels of a head turned by time, height and width: height and width a third each,
    rounded down to even, time the rest (less one where head_dim is odd)."""
    side = 2 * (head_dim // 6)
    return (head_dim - head_dim % 2 - 2 * side, side, side)


def video_positions(video_shape: Sequence[int], device=None) -> Tensor:
    """(t, h, w) of every token of a video grid, [T*H*W, 3] int32, in token order."""
    t, h, w = (torch.arange(int(n), dtype=torch.int32, device=device) for n in video_shape)
    return torch.stack(torch.meshgrid(t, h, w, indexing="ij"), -1).reshape(-1, 3)


def _device_index(*ts: Optional[Tensor]) -> int:
    """The one device that all tensors are on."""
    index = -1
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("megaslide_amd kernels run on ROCm devices only; got a tensor on "
                               f"{t.device} (there is no CPU implementation)")
        i = t.get_device()
        if index < 0:
            index = i
        elif i != index:
            raise RuntimeError(f"megaslide_amd: tensors on different devices ({index}, {i})")
    return index


def _rows(t: Tensor, name: str) -> Tuple[Tensor, int]:
    """``t`` ([N, D] or [B, N, D]) with unit channel stride and one stride between tokens, and
    that stride; a copy where its own layout is another."""
    shape = t.shape
    if len(shape) not in (2, 3):
        raise ValueError(f"{name} must be [N, D] or [B, N, D], got {tuple(shape)}")
    D = shape[-1]
    if t.is_contiguous() or t.numel() == 0:
        return t, max(D, 1)
    if t.stride(-1) == 1 or D == 1:
        if t.dim() == 2 or t.shape[0] == 1:
            s = t.stride(-2) if t.shape[-2] > 1 else D
        elif t.shape[1] == 1:
            s = t.stride(0)
        else:
            s = t.stride(1) if t.stride(0) == t.shape[1] * t.stride(1) else 0
        if s >= D:
            return t, s
    return t.contiguous(), D


def _split_heads(t: Tensor, heads: int, name: str) -> int:
    if heads < 1:
        raise ValueError(f"number of heads must be positive, got {heads}")
    if t.shape[-1] % heads != 0 or t.shape[-1] == 0:
        raise ValueError(f"{name}: {t.shape[-1]} channels do not split into {heads} heads")
    return t.shape[-1] // heads


# ---------------------------------------------------------------------------
# rotation, norm
# ---------------------------------------------------------------------------

_Int4, _Int3 = ctypes.c_int32 * 4, ctypes.c_int32 * 3
_NO_GRID = _Int3(0, 0, 0)


class _RopeCall:
    """Validated arguments of one rotation; ``head``, ``tail``: its C descriptor before and behind
    the strides."""

    __slots__ = ("index", "weights", "pos", "head", "tail")

    def __init__(self, what, q, k, wq, wk, positions, num_heads, num_kv_heads, axes, theta, eps,
                 interleaved, norm):
        on_grid = not isinstance(positions, Tensor)
        self.index = _device_index(q, k, wq, wk, None if on_grid else positions)
        hd = _split_heads(q, num_heads, what)
        shape, dt = q.shape, q.dtype
        n = shape[-2] if len(shape) > 1 else 0
        if k is not None:
            if k.dtype != dt:
                raise TypeError(f"{what}: k is {k.dtype}, q is {dt}")
            if k.shape[:-1] != shape[:-1] or k.shape[-1] != num_kv_heads * hd:
                raise ValueError(f"{what}: k must be {(*shape[:-1], num_kv_heads * hd)}, got "
                                 f"{tuple(k.shape)}")
        wdt = None
        for name, w in (("q_weight", wq), ("k_weight", wk)):
            if w is None:
                continue
            if w.shape != (hd,):
                raise ValueError(f"{what}: {name} must be {(hd,)}, got {tuple(w.shape)}")
            if w.dtype != torch.float32 and w.dtype != dt:
                raise TypeError(f"{what}: {name} is {w.dtype}, must be float32 or {dt}")
            if wdt is not None and w.dtype != wdt:
                raise TypeError(f"{what}: q_weight and k_weight differ in dtype")
            wdt = w.dtype
        self.weights = (None if wq is None else wq.contiguous(),
                        None if wk is None else wk.contiguous())
        if on_grid:
            grid = tuple(int(s) for s in positions)
            if len(grid) != 3 or min(grid) < 0 or math.prod(grid) != n:
                raise ValueError(f"{what}: a grid (T, H, W) of {n} tokens, got {grid}")
            self.pos, n_axes, rows, pdt, grid = None, 3, n, _lib.POS_GRID, _Int3(*grid)
        else:
            pdt = _lib.POS_DTYPES.get(positions.dtype)
            if pdt is None:
                raise TypeError(f"{what}: positions are {positions.dtype}, must be one of "
                                f"{[str(t) for t in _lib.POS_DTYPES]}")
            if positions.requires_grad:
                raise ValueError(f"{what}: positions have no gradient")
            ps = positions.shape
            if len(ps) < 2 or (ps[:-1] != (n,) and ps[:-1] != shape[:-1]):
                raise ValueError(f"{what}: positions must be [{n}, axes] or "
                                 f"{(*shape[:-1], 'axes')}, got {tuple(ps)}")
            self.pos, n_axes, grid = positions.contiguous(), ps[-1], _NO_GRID
            rows = n if len(ps) == 2 else n * ps[0]
        if axes is None:
            if n_axes != 1 and n_axes != 3:
                raise ValueError(f"{what}: axes must be given for {n_axes} columns of positions")
            axes = (hd - hd % 2,) if n_axes == 1 else video_axes(hd)
        axes = tuple(int(d) for d in axes)
        if len(axes) != n_axes or not 1 <= n_axes <= 4:
            raise ValueError(f"{what}: {len(axes)} axes, positions have {n_axes} columns (1 to 4)")
        if any(d < 0 or d % 2 for d in axes) or sum(axes) > hd:
            raise ValueError(f"{what}: axes {axes} must be even and at most {hd} channels together")
        self.head = (q.numel() // shape[-1], rows)
        self.tail = (float(theta), num_heads, 0 if k is None else num_kv_heads, hd,
                     _lib.dtype_code(dt), 0 if wdt is None else _lib.dtype_code(wdt), pdt, n_axes,
                     _Int4(*axes), 1 if interleaved else 0, 1 if norm else 0, float(eps), grid)

    def forward(self, q, k):
        qr, qs = _rows(q, "q")
        kr, ks = (None, 0) if k is None else _rows(k, "k")
        yq, yk = q.new_empty(q.shape), None if k is None else k.new_empty(k.shape)
        wq, wk = self.weights
        desc = _lib.QkRopeDesc(*self.head, qs, ks, *self.tail)
        ptr = _lib.ptr
        _lib.launch(_lib.load().msd_qk_rope_fwd, "qk_rope_fwd", self.index, ctypes.byref(desc),
                    qr.data_ptr(), ptr(kr), ptr(wq), ptr(wk), ptr(self.pos), yq.data_ptr(),
                    ptr(yk))
        return yq, yk

    def backward(self, q, k, dyq, dyk, want_dw):
        """Gradients of q, k and (with the norm, where wanted) of the weights."""
        dt = dyq.dtype
        dyq = dyq.contiguous()
        dyk = None if dyk is None else dyk.to(dt).contiguous()
        qr, qs = (None, dyq.shape[-1]) if q is None else _rows(q, "q")
        kr, ks = (None, 0 if dyk is None else dyk.shape[-1]) if k is None else _rows(k, "k")
        dq, dk = dyq.new_empty(dyq.shape), None if dyk is None else dyk.new_empty(dyk.shape)
        wq, wk = self.weights
        dwq = torch.empty_like(wq) if wq is not None and want_dw[0] else None
        dwk = torch.empty_like(wk) if wk is not None and want_dw[1] else None
        desc = _lib.QkRopeDesc(*self.head, qs, ks, *self.tail)
        lib, ptr, d = _lib.load(), _lib.ptr, ctypes.byref(desc)
        need = lib.msd_qk_rope_bwd_workspace_size(d)
        ws = dyq.new_empty(need, dtype=torch.uint8) if need else None
        _lib.launch(lib.msd_qk_rope_bwd, "qk_rope_bwd", self.index, d, ptr(qr), ptr(kr), ptr(wq),
                    ptr(wk), ptr(self.pos), dyq.data_ptr(), ptr(dyk), dq.data_ptr(), ptr(dk),
                    ptr(dwq), ptr(dwk), ptr(ws), need)
        return dq, dk, dwq, dwk


class AxialRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, call):
        y = call.forward(x, None)[0]
        ctx.call, ctx.dtype = call, x.dtype
        ctx.save_for_backward(call.pos)
        call.pos = None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        call = ctx.call
        (call.pos,) = ctx.saved_tensors
        try:
            return call.backward(None, None, dy.to(ctx.dtype), None, (False, False))[0], None
        finally:
            call.pos = None


class QkNormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, call):
        ys = call.forward(q, k)
        ctx.call = call
        ctx.save_for_backward(q, k, *call.weights, call.pos)
        call.weights = call.pos = None
        return ys

    @staticmethod
    @once_differentiable
    def backward(ctx, dyq, dyk):
        call = ctx.call
        q, k, wq, wk, call.pos = ctx.saved_tensors
        call.weights = (wq, wk)
        try:
            return (*call.backward(q, k, dyq.to(q.dtype), dyk, ctx.needs_input_grad[2:4]), None)
        finally:
            call.weights = call.pos = None


def axial_rope(x: Tensor, positions: Positions, num_heads: int,
               axes: Optional[Sequence[int]] = None, theta: float = 10000.0,
               interleaved: bool = False) -> Tensor:
    """Rotary positions with one or several axes, for queries or keys x [B, N, D] or [N, D].

    Each head's channels are split among the axes (``axes``: even counts, at most head_dim
    together; channels behind them pass through unchanged).  Pair i of axis a, of d_a channels,
    turns by positions[n, a] * theta^(-2 i / d_a); pairs are (2i, 2i+1) of the axis's channels
    (``interleaved``) or (i, i + d_a/2).  ``positions``: [N, axes] or [B, N, axes] of int32,
    int64, float32 or float64, without gradient, or a video grid (T, H, W) of N tokens.  ``axes``
    None: all channels for one axis, ``video_axes(head_dim)`` for three.  Angles are held in 64
    bits.  Differentiable in x, once.
    """
    call = _RopeCall("axial_rope", x, None, None, None, positions, int(num_heads), 0, axes, theta,
                     0.0, interleaved, False)
    if torch.is_grad_enabled() and x.requires_grad:
        return AxialRopeFunction.apply(x, call)
    return call.forward(x, None)[0]


def qk_norm_rope(q: Tensor, k: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor],
                 positions: Positions, num_heads: int, num_kv_heads: Optional[int] = None,
                 axes: Optional[Sequence[int]] = None, theta: float = 10000.0, eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[Tensor, Tensor]:
    """RMS norm of each head of q [B, N, D] (or [N, D]) and k [B, N, num_kv_heads * head_dim],
    times the weight of its channel, and the rotation of ``axial_rope``, in one pass.

    q_weight, k_weight: [head_dim] (None: ones), float32 or the dtype of q.  q and k may be views
    of one fused projection's output.  The arithmetic is fp32 and is rounded once.
    Differentiable in q, k and the weights, once; the weights' gradients are summed in a fixed
    order.
    """
    num_kv_heads = int(num_heads if num_kv_heads is None else num_kv_heads)
    call = _RopeCall("qk_norm_rope", q, k, q_weight, k_weight, positions, int(num_heads),
                     num_kv_heads, axes, theta, eps, interleaved, True)
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return QkNormRopeFunction.apply(q, k, q_weight, k_weight, call)
    return call.forward(q, k)


# ---------------------------------------------------------------------------
# attention over packed sequences
# ---------------------------------------------------------------------------

class _AttnCall:
    """Validated arguments of one packed attention and its C descriptor."""

    __slots__ = ("index", "q", "k", "v", "cu_q", "cu_k", "heads", "desc")

    def __init__(self, q, k, v, cu_q, cu_k, num_heads, num_kv_heads, causal, scale):
        what = "packed_attention"
        self.index = _device_index(q, k, v, cu_q, cu_k)
        hd = _split_heads(q, num_heads, what)
        if num_kv_heads < 1 or num_heads % num_kv_heads != 0:
            raise ValueError(f"{what}: num_heads={num_heads} must be a multiple of "
                             f"num_kv_heads={num_kv_heads}")
        qsh, ksh, dt = q.shape, k.shape, q.dtype
        for name, t in (("k", k), ("v", v)):
            if t.dtype != dt:
                raise TypeError(f"{what}: {name} is {t.dtype}, q is {dt}")
            if len(t.shape) != len(qsh) or t.shape[-1] != num_kv_heads * hd:
                raise ValueError(f"{what}: {name} must have {num_kv_heads * hd} channels and as "
                                 f"many dimensions as q, got {tuple(t.shape)}")
        if ksh != v.shape:
            raise ValueError(f"{what}: k {tuple(ksh)} and v {tuple(v.shape)} differ")
        self.q, qs = _rows(q, "q")
        self.k, ks = _rows(k, "k")
        self.v, vs = _rows(v, "v")
        self.cu_q, self.cu_k = cu_q, cu_q if cu_k is None else cu_k
        if cu_q is None:
            if cu_k is not None:
                raise ValueError(f"{what}: cu_seqlens_k without cu_seqlens")
            seqs = 1
            if len(qsh) == 3:
                seqs = qsh[0]
                if ksh[0] != seqs:
                    raise ValueError(f"{what}: batches {seqs} of q and {ksh[0]} of k")
        else:
            if len(qsh) != 2:
                raise ValueError(f"{what}: packed sequences are [N, D], got {tuple(qsh)}")
            for name, c in (("cu_seqlens", cu_q), ("cu_seqlens_k", self.cu_k)):
                if c.dtype != torch.int32 or c.dim() != 1 or c.numel() < 2 or not c.is_contiguous():
                    raise ValueError(f"{what}: {name} must be contiguous int32 of sequences + 1 "
                                     f"entries, got {c.dtype} {tuple(c.shape)}")
            seqs = cu_q.numel() - 1
            if cu_k is None:
                if qsh[0] != ksh[0]:
                    raise ValueError(f"{what}: q has {qsh[0]} rows and k {ksh[0]}; give "
                                     "cu_seqlens_k")
            elif cu_k.numel() != seqs + 1:
                raise ValueError(f"{what}: {seqs} sequences of q and {cu_k.numel() - 1} of k")
        self.heads = num_heads
        self.desc = _lib.AttnDesc(
            q.numel() // qsh[-1], k.numel() // ksh[-1], qs, ks, vs, max(seqs, 1), num_heads,
            num_kv_heads, hd, _lib.dtype_code(dt), 1 if causal else 0,
            1.0 / math.sqrt(hd) if scale is None else float(scale))

    def take(self):
        """The call's tensors, which it then holds no more (autograd saves them)."""
        tensors = (self.q, self.k, self.v, self.cu_q, self.cu_k)
        self.q = self.k = self.v = self.cu_q = self.cu_k = None
        return tensors

    def give(self, tensors) -> None:
        """Those tensors again, whose layout may be another one (hooks on saved tensors move and
        copy them)."""
        q, k, v, self.cu_q, self.cu_k = tensors
        self.q, self.desc.q_stride = _rows(q, "q")
        self.k, self.desc.k_stride = _rows(k, "k")
        self.v, self.desc.v_stride = _rows(v, "v")

    def forward(self, want_lse: bool, want_rest: bool = False):
        """out, lse and what rounding took from out (bf16, for the backward), as wanted."""
        q, ptr = self.q, _lib.ptr
        out = q.new_empty(q.shape)
        rest = q.new_empty(q.shape) if want_rest and q.dtype == torch.bfloat16 else None
        lse = q.new_empty((*q.shape[:-1], self.heads), dtype=torch.float32) if want_lse else None
        lib, d = _lib.load(), ctypes.byref(self.desc)
        need = lib.msd_attn_fwd_workspace_size(d)
        ws = q.new_empty(need, dtype=torch.uint8) if need else None
        _lib.launch(lib.msd_attn_fwd, "attn_fwd", self.index, d, q.data_ptr(), self.k.data_ptr(),
                    self.v.data_ptr(), ptr(self.cu_q), ptr(self.cu_k), out.data_ptr(), ptr(rest),
                    ptr(lse), ptr(ws), need)
        return out, lse, rest

    def backward(self, out, lse, rest, dout, dlse):
        q, ptr = self.q, _lib.ptr
        out, lse, dout = out.contiguous(), lse.contiguous(), dout.to(q.dtype).contiguous()
        rest = None if rest is None or rest.numel() == 0 else rest.contiguous()
        dlse = None if dlse is None else dlse.to(torch.float32).contiguous()
        dq, dk, dv = (t.new_empty(t.shape) for t in (q, self.k, self.v))
        lib, d = _lib.load(), ctypes.byref(self.desc)
        need = lib.msd_attn_bwd_workspace_size(d)
        ws = q.new_empty(max(need, 16), dtype=torch.uint8)
        _lib.launch(lib.msd_attn_bwd, "attn_bwd", self.index, d, q.data_ptr(), self.k.data_ptr(),
                    self.v.data_ptr(), ptr(self.cu_q), ptr(self.cu_k), out.data_ptr(),
                    ptr(rest), dout.data_ptr(), lse.data_ptr(), ptr(dlse), dq.data_ptr(),
                    dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), need)
        return dq, dk, dv


# As the deformable core, a torch.library custom operator, so that selective checkpointing can
# keep its outputs and torch.compile takes it as one opaque op.

@torch.library.custom_op("megaslide::packed_attention", mutates_args=(), device_types="cuda")
def _attn_fwd_op(q: Tensor, k: Tensor, v: Tensor, cu_seqlens: Optional[Tensor],
                 cu_seqlens_k: Optional[Tensor], num_heads: int, num_kv_heads: int, causal: bool,
                 scale: Optional[float]) -> Tuple[Tensor, Tensor, Tensor]:
    """out like q, lse [..., num_heads] (fp32) and what rounding took from out (bf16, else
    empty), which keeps the backward's sums of dout * out exact."""
    out, lse, rest = _AttnCall(q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, causal,
                               scale).forward(want_lse=True, want_rest=True)
    return out, lse, q.new_empty((0,)) if rest is None else rest


@_attn_fwd_op.register_fake
def _(q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, causal, scale):
    return (q.new_empty(q.shape),
            q.new_empty((*q.shape[:-1], num_heads), dtype=torch.float32),
            q.new_empty(q.shape if q.dtype == torch.bfloat16 else (0,)))


@torch.library.custom_op("megaslide::packed_attention_bwd", mutates_args=(), device_types="cuda")
def _attn_bwd_op(q: Tensor, k: Tensor, v: Tensor, cu_seqlens: Optional[Tensor],
                 cu_seqlens_k: Optional[Tensor], out: Tensor, lse: Tensor, rest: Tensor,
                 dout: Tensor, dlse: Optional[Tensor], num_heads: int, num_kv_heads: int,
                 causal: bool, scale: Optional[float]) -> Tuple[Tensor, Tensor, Tensor]:
    """dq, dk, dv."""
    return _AttnCall(q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, causal,
                     scale).backward(out, lse, rest, dout, dlse)


@_attn_bwd_op.register_fake
def _(q, k, v, cu_seqlens, cu_seqlens_k, out, lse, rest, dout, dlse, num_heads, num_kv_heads,
      causal, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _attn_setup(ctx, inputs, output):
    ctx.args = inputs[5:]
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(*inputs[:5], *output)


def _attn_backward(ctx, dout, dlse, drest):
    q, k, v, cu, cu_k, out, lse, rest = ctx.saved_tensors
    if dout is None:
        dout = torch.zeros_like(out)
    return (*_attn_bwd_op(q, k, v, cu, cu_k, out, lse, rest, dout, dlse,
                          *ctx.args),) + (None,) * 6


_attn_fwd_op.register_autograd(_attn_backward, setup_context=_attn_setup)


class PackedAttentionFunction(torch.autograd.Function):
    """The custom operator's forward and backward without the dispatcher between, which would
    cost a small training call several times its kernels' time; for calls that no dispatch mode
    (selective checkpointing) and no compiler has to see."""

    @staticmethod
    def forward(ctx, q, k, v, call):
        out, lse, rest = call.forward(want_lse=True, want_rest=True)
        ctx.call = call
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*call.take(), out, lse, rest)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlse):
        *tensors, out, lse, rest = ctx.saved_tensors
        if dout is None:
            dout = torch.zeros_like(out)
        call = ctx.call
        call.give(tensors)
        try:
            return (*call.backward(out, lse, rest, dout, dlse), None)
        finally:
            call.take()


def packed_attention(q: Tensor, k: Tensor, v: Tensor, num_heads: int,
                     num_kv_heads: Optional[int] = None, cu_seqlens: Optional[Tensor] = None,
                     cu_seqlens_k: Optional[Tensor] = None, causal: bool = False,
                     scale: Optional[float] = None, return_lse: bool = False):
    """softmax(scale q k^T + mask) v of each sequence and head.

    Packed: q [N, num_heads * head_dim], k and v [M, num_kv_heads * head_dim]; sequence s has the
    rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 of q and those of ``cu_seqlens_k`` (default: the
    same) of k and v.  The offsets are int32 on the device and are read there (nothing
    synchronises); they begin with 0, do not fall and end at most at N (M).  Rows behind the last
    sequence have out 0 and no gradient.  Without offsets: [B, N, D] and [B, M, D], B sequences
    of equal length, or [N, D], one sequence.

    Query head h reads key head h // (num_heads // num_kv_heads).  ``causal``: query i of n sees
    the keys j <= i + m - n (the last query sees the last key, so that one new token over a
    cache sees all of it).  A query that sees no key (or none with a score above -inf) has out 0 and
    lse -inf.  What a query does not see does not change its result, infinities and NaN there
    included.  ``scale``: default 1 / sqrt(head_dim); positive.  head_dim up to 128.

    Returns out like q (and lse, the log-sum-exp of the scaled scores, fp32 [..., num_heads]);
    both are differentiable, once.  Gradients are summed without atomics, in a fixed order.
    """
    num_heads = int(num_heads)
    num_kv_heads = int(num_heads if num_kv_heads is None else num_kv_heads)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        if not torch.compiler.is_compiling() and torch._C._len_torch_dispatch_stack() == 0:
            out, lse = PackedAttentionFunction.apply(q, k, v, _AttnCall(
                q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, causal, scale))
            return (out, lse) if return_lse else out
        out, lse, _ = torch.ops.megaslide.packed_attention(
            q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, bool(causal),
            None if scale is None else float(scale))
    else:
        out, lse, _ = _AttnCall(q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, causal,
                                scale).forward(want_lse=return_lse)
    return (out, lse) if return_lse else out
