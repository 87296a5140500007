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
from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _require_device

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


def _rows(t: Tensor, name: str) -> Tuple[Tensor, int]:
    """``t`` ([N, D] or [B, N, D]) with unit channel stride and one stride between tokens, and
    that stride; a copy where its own layout is another."""
    if t.dim() not in (2, 3):
        raise ValueError(f"{name} must be [N, D] or [B, N, D], got {tuple(t.shape)}")
    D = t.shape[-1]
    if t.numel() == 0 or t.is_contiguous():
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

class _RopeCall:
    """Validated arguments of one rotation and its C descriptor."""

    def __init__(self, what, q, k, weights, positions, num_heads, num_kv_heads, axes, theta, eps,
                 interleaved, norm):
        ts = [q, k, *weights]
        if isinstance(positions, Tensor):
            ts.append(positions)
        self.dev = _require_device(*ts)
        hd = _split_heads(q, num_heads, what)
        tokens = q.numel() // q.shape[-1]
        self.shape = q.shape[:-1]
        if k is not None:
            if k.dtype != q.dtype:
                raise TypeError(f"{what}: k is {k.dtype}, q is {q.dtype}")
            if k.shape[:-1] != q.shape[:-1] or k.shape[-1] != num_kv_heads * hd:
                raise ValueError(f"{what}: k must be {(*q.shape[:-1], num_kv_heads * hd)}, got "
                                 f"{tuple(k.shape)}")
        self.weights, wdt = [], torch.float32
        for name, w in zip(("q_weight", "k_weight"), weights):
            if w is None:
                self.weights.append(None)
                continue
            if w.shape != (hd,):
                raise ValueError(f"{what}: {name} must be {(hd,)}, got {tuple(w.shape)}")
            if w.dtype not in (torch.float32, q.dtype):
                raise TypeError(f"{what}: {name} is {w.dtype}, must be float32 or {q.dtype}")
            self.weights.append(w.contiguous())
            wdt = w.dtype
        if len({w.dtype for w in self.weights if w is not None}) > 1:
            raise TypeError(f"{what}: q_weight and k_weight differ in dtype")
        self.wdt = wdt
        grid = (0, 0, 0)
        n = q.shape[-2]
        if isinstance(positions, Tensor):
            if positions.dtype not in _lib.POS_DTYPES:
                raise TypeError(f"{what}: positions are {positions.dtype}, must be one of "
                                f"{[str(t) for t in _lib.POS_DTYPES]}")
            if positions.requires_grad:
                raise ValueError(f"{what}: positions have no gradient")
            if positions.dim() < 1 or positions.shape[:-1] not in ((n,), tuple(self.shape)):
                raise ValueError(f"{what}: positions must be [{n}, axes] or "
                                 f"{(*self.shape, 'axes')}, got {tuple(positions.shape)}")
            self.pos, n_axes = positions.contiguous(), positions.shape[-1]
            rows, pdt = positions.numel() // max(n_axes, 1), _lib.POS_DTYPES[positions.dtype]
        else:
            grid = tuple(int(s) for s in positions)
            if len(grid) != 3 or min(grid) < 0 or math.prod(grid) != n:
                raise ValueError(f"{what}: a grid (T, H, W) of {n} tokens, got {grid}")
            self.pos, n_axes, rows, pdt = None, 3, n, _lib.POS_GRID
        if axes is None:
            axes = {1: (hd - hd % 2,), 3: video_axes(hd)}.get(n_axes)
            if axes is None:
                raise ValueError(f"{what}: axes must be given for {n_axes} columns of positions")
        axes = tuple(int(d) for d in axes)
        if len(axes) != n_axes or not 1 <= n_axes <= 4:
            raise ValueError(f"{what}: {len(axes)} axes, positions have {n_axes} columns (1 to 4)")
        if any(d < 0 or d % 2 for d in axes) or sum(axes) > hd:
            raise ValueError(f"{what}: axes {axes} must be even and at most {hd} channels together")
        self.hd, self.tokens, self.heads = hd, tokens, (num_heads, 0 if k is None else num_kv_heads)
        self.args = dict(theta=float(theta), dtype=_lib.dtype_code(q.dtype),
                         weight_dtype=_lib.dtype_code(wdt), pos_dtype=pdt, n_axes=n_axes,
                         axis_dims=(ctypes.c_int32 * 4)(*axes), interleaved=int(bool(interleaved)),
                         norm=int(norm), eps=float(eps), grid=(ctypes.c_int32 * 3)(*grid),
                         pos_rows=rows)

    def desc(self, qs: int, ks: int) -> _lib.QkRopeDesc:
        return _lib.QkRopeDesc(tokens=self.tokens, q_stride=qs, k_stride=ks,
                               q_heads=self.heads[0], k_heads=self.heads[1], head_dim=self.hd,
                               **self.args)

    def empty(self, like: Tensor) -> Tensor:
        return torch.empty(like.shape, dtype=like.dtype, device=self.dev)

    def forward(self, q, k):
        qr, qs = _rows(q, "q")
        kr, ks = (None, 0) if k is None else _rows(k, "k")
        yq, yk = self.empty(q), None if k is None else self.empty(k)
        wq, wk = self.weights
        desc = self.desc(qs, ks)
        lib = _lib.load()
        with torch.cuda.device(self.dev):
            _lib.check(lib.msd_qk_rope_fwd(
                ctypes.byref(desc), qr.data_ptr(), _lib.ptr(kr), _lib.ptr(wq), _lib.ptr(wk),
                _lib.ptr(self.pos), yq.data_ptr(), _lib.ptr(yk), _lib.stream_handle(self.dev)),
                "qk_rope_fwd")
        return yq, yk

    def backward(self, q, k, dyq, dyk, want_dw):
        """Gradients of q, k and (with the norm, where wanted) of the weights."""
        dt = dyq.dtype
        dyq = dyq.contiguous()
        dyk = None if dyk is None else dyk.to(dt).contiguous()
        qr, qs = (None, dyq.shape[-1]) if q is None else _rows(q, "q")
        kr, ks = (None, 0 if dyk is None else dyk.shape[-1]) if k is None else _rows(k, "k")
        dq, dk = self.empty(dyq), None if dyk is None else self.empty(dyk)
        dw = [None if w is None or not want else torch.empty_like(w)
              for w, want in zip(self.weights, want_dw)]
        wq, wk = self.weights
        desc = self.desc(qs, ks)
        lib = _lib.load()
        need = lib.msd_qk_rope_bwd_workspace_size(ctypes.byref(desc))
        ws = torch.empty(need, dtype=torch.uint8, device=self.dev) if need else None
        with torch.cuda.device(self.dev):
            _lib.check(lib.msd_qk_rope_bwd(
                ctypes.byref(desc), _lib.ptr(qr), _lib.ptr(kr), _lib.ptr(wq), _lib.ptr(wk),
                _lib.ptr(self.pos), dyq.data_ptr(), _lib.ptr(dyk), dq.data_ptr(), _lib.ptr(dk),
                _lib.ptr(dw[0]), _lib.ptr(dw[1]), _lib.ptr(ws), need,
                _lib.stream_handle(self.dev)), "qk_rope_bwd")
        return dq, dk, dw[0], dw[1]


class AxialRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, call):
        ctx.call = call
        ctx.dtype = x.dtype
        return call.forward(x, None)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return ctx.call.backward(None, None, dy.to(ctx.dtype), None, (False, False))[0], None


class QkNormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, call):
        ctx.call = call
        ctx.save_for_backward(q, k)
        return call.forward(q, k)

    @staticmethod
    @once_differentiable
    def backward(ctx, dyq, dyk):
        q, k = ctx.saved_tensors
        return (*ctx.call.backward(q, k, dyq.to(q.dtype), dyk, ctx.needs_input_grad[2:4]), None)


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
    call = _RopeCall("axial_rope", x, None, (None, None), positions, int(num_heads), 0, axes, theta,
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
    call = _RopeCall("qk_norm_rope", q, k, (q_weight, k_weight), positions, int(num_heads),
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

    def __init__(self, q, k, v, cu_q, cu_k, num_heads, num_kv_heads, causal, scale):
        what = "packed_attention"
        self.dev = _require_device(q, k, v, cu_q, cu_k)
        hd = _split_heads(q, num_heads, what)
        if num_kv_heads < 1 or num_heads % num_kv_heads != 0:
            raise ValueError(f"{what}: num_heads={num_heads} must be a multiple of "
                             f"num_kv_heads={num_kv_heads}")
        for name, t in (("k", k), ("v", v)):
            if t.dtype != q.dtype:
                raise TypeError(f"{what}: {name} is {t.dtype}, q is {q.dtype}")
            if t.dim() != q.dim() or t.shape[-1] != num_kv_heads * hd:
                raise ValueError(f"{what}: {name} must have {num_kv_heads * hd} channels and as "
                                 f"many dimensions as q, got {tuple(t.shape)}")
        if k.shape != v.shape:
            raise ValueError(f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
        self.q, qs = _rows(q, "q")
        self.k, ks = _rows(k, "k")
        self.v, vs = _rows(v, "v")
        self.cu_q, self.cu_k = cu_q, cu_q if cu_k is None else cu_k
        if cu_q is None:
            if cu_k is not None:
                raise ValueError(f"{what}: cu_seqlens_k without cu_seqlens")
            if q.dim() == 3:
                if k.shape[0] != q.shape[0]:
                    raise ValueError(f"{what}: batches {q.shape[0]} of q and {k.shape[0]} of k")
                seqs = q.shape[0]
            else:
                seqs = 1
        else:
            if q.dim() != 2:
                raise ValueError(f"{what}: packed sequences are [N, D], got {tuple(q.shape)}")
            for name, c in (("cu_seqlens", cu_q), ("cu_seqlens_k", self.cu_k)):
                if c.dtype != torch.int32 or c.dim() != 1 or c.numel() < 2 or not c.is_contiguous():
                    raise ValueError(f"{what}: {name} must be contiguous int32 of sequences + 1 "
                                     f"entries, got {c.dtype} {tuple(c.shape)}")
            seqs = cu_q.numel() - 1
            if self.cu_k.numel() != seqs + 1:
                raise ValueError(f"{what}: {seqs} sequences of q and {self.cu_k.numel() - 1} of k")
            if cu_k is None and q.shape[0] != k.shape[0]:
                raise ValueError(f"{what}: q has {q.shape[0]} rows and k {k.shape[0]}; give "
                                 "cu_seqlens_k")
        self.shape, self.hd, self.heads = q.shape, hd, num_heads
        self.desc = _lib.AttnDesc(
            q.numel() // q.shape[-1], k.numel() // k.shape[-1], qs, ks, vs, max(seqs, 1), num_heads,
            num_kv_heads, hd, _lib.dtype_code(q.dtype), int(bool(causal)),
            1.0 / math.sqrt(hd) if scale is None else float(scale))

    def forward(self, want_lse: bool):
        q = self.q
        out = torch.empty(self.shape, dtype=q.dtype, device=self.dev)
        lse = (torch.empty((*self.shape[:-1], self.heads), dtype=torch.float32, device=self.dev)
               if want_lse else None)
        lib = _lib.load()
        d = ctypes.byref(self.desc)
        need = lib.msd_attn_fwd_workspace_size(d)
        ws = torch.empty(need, dtype=torch.uint8, device=self.dev) if need else None
        with torch.cuda.device(self.dev):
            _lib.check(lib.msd_attn_fwd(
                d, q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), _lib.ptr(self.cu_q),
                _lib.ptr(self.cu_k), out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), need,
                _lib.stream_handle(self.dev)), "attn_fwd")
        return out, lse

    def backward(self, out, lse, dout, dlse):
        dt = self.q.dtype
        out, lse, dout = out.contiguous(), lse.contiguous(), dout.to(dt).contiguous()
        dlse = None if dlse is None else dlse.to(torch.float32).contiguous()
        dq, dk, dv = (torch.empty(t.shape, dtype=dt, device=self.dev)
                      for t in (self.q, self.k, self.v))
        lib = _lib.load()
        d = ctypes.byref(self.desc)
        need = lib.msd_attn_bwd_workspace_size(d)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=self.dev)
        with torch.cuda.device(self.dev):
            _lib.check(lib.msd_attn_bwd(
                d, self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), _lib.ptr(self.cu_q),
                _lib.ptr(self.cu_k), out.data_ptr(), dout.data_ptr(), lse.data_ptr(),
                _lib.ptr(dlse), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), need,
                _lib.stream_handle(self.dev)), "attn_bwd")
        return dq, dk, dv


# As the deformable core, a torch.library custom operator, so that selective checkpointing can
# keep its outputs and torch.compile takes it as one opaque op.

@torch.library.custom_op("megaslide::packed_attention", mutates_args=(), device_types="cuda")
def _attn_fwd_op(q: Tensor, k: Tensor, v: Tensor, cu_seqlens: Optional[Tensor],
                 cu_seqlens_k: Optional[Tensor], num_heads: int, num_kv_heads: int, causal: bool,
                 scale: Optional[float]) -> Tuple[Tensor, Tensor]:
    """out like q and lse [..., num_heads] (fp32)."""
    return _AttnCall(q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, causal,
                     scale).forward(want_lse=True)


@_attn_fwd_op.register_fake
def _(q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, causal, scale):
    return (q.new_empty(q.shape),
            q.new_empty((*q.shape[:-1], num_heads), dtype=torch.float32))


@torch.library.custom_op("megaslide::packed_attention_bwd", mutates_args=(), device_types="cuda")
def _attn_bwd_op(q: Tensor, k: Tensor, v: Tensor, cu_seqlens: Optional[Tensor],
                 cu_seqlens_k: Optional[Tensor], out: Tensor, lse: Tensor, dout: Tensor,
                 dlse: Optional[Tensor], num_heads: int, num_kv_heads: int, causal: bool,
                 scale: Optional[float]) -> Tuple[Tensor, Tensor, Tensor]:
    """dq, dk, dv."""
    return _AttnCall(q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, causal,
                     scale).backward(out, lse, dout, dlse)


@_attn_bwd_op.register_fake
def _(q, k, v, cu_seqlens, cu_seqlens_k, out, lse, dout, dlse, num_heads, num_kv_heads, causal,
      scale):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _attn_setup(ctx, inputs, output):
    ctx.args = inputs[5:]
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(*inputs[:5], *output)


def _attn_backward(ctx, dout, dlse):
    q, k, v, cu, cu_k, out, lse = ctx.saved_tensors
    if dout is None:
        dout = torch.zeros_like(out)
    return (*_attn_bwd_op(q, k, v, cu, cu_k, out, lse, dout, dlse, *ctx.args),) + (None,) * 6


_attn_fwd_op.register_autograd(_attn_backward, setup_context=_attn_setup)


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
    cache sees all of it).  A query that sees no key has out 0 and lse -inf.  What a query does
    not see does not change its result, infinities and NaN there included.  ``scale``: default
    1 / sqrt(head_dim); positive.  head_dim up to 128.

    Returns out like q (and lse, the log-sum-exp of the scaled scores, fp32 [..., num_heads]);
    both are differentiable, once.  Gradients are summed without atomics, in a fixed order.
    """
    num_heads = int(num_heads)
    num_kv_heads = int(num_heads if num_kv_heads is None else num_kv_heads)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
        out, lse = torch.ops.megaslide.packed_attention(
            q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, bool(causal),
            None if scale is None else float(scale))
    else:
        out, lse = _AttnCall(q, k, v, cu_seqlens, cu_seqlens_k, num_heads, num_kv_heads, causal,
                             scale).forward(want_lse=return_lse)
    return (out, lse) if return_lse else out
