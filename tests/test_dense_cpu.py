"""Checks of the dense attention operators that need no GPU: the C ABI refuses bad arguments with
a status and a message before any device work, sizes of workspaces, helpers of the host side."""

import ctypes
import os

import pytest
import torch

from megaslide_amd import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH),
                                reason="HIP library not built (python -m megaslide_amd.csrc.build)")


def rope_desc(**kw):
    d = dict(tokens=24, pos_rows=24, q_stride=256, k_stride=128, theta=1e4, q_heads=4, k_heads=2,
             head_dim=64, dtype=0, weight_dtype=0, pos_dtype=0, n_axes=3, axis_dims=(24, 20, 20, 0),
             interleaved=0, norm=1, eps=1e-6, grid=(0, 0, 0))
    d.update(kw)
    d["axis_dims"] = (ctypes.c_int32 * 4)(*d["axis_dims"])
    d["grid"] = (ctypes.c_int32 * 3)(*d["grid"])
    return _lib.QkRopeDesc(**d)


def rope_fwd(desc, ptrs=(16, 16, 16, 16, 16, 16, 16)):
    return _lib.load().msd_qk_rope_fwd(None if desc is None else ctypes.byref(desc), *ptrs, None)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(tokens=-1), -1, b"sizes"),
    (dict(pos_rows=0), -1, b"sizes"),
    (dict(q_heads=0), -1, b"heads"),
    (dict(k_heads=-1), -1, b"heads"),
    (dict(head_dim=1), -2, b"head_dim"),
    (dict(head_dim=258, q_stride=2000, k_stride=2000), -2, b"head_dim"),
    (dict(dtype=2), -2, b"dtype"),
    (dict(weight_dtype=1), -2, b"weight_dtype"),     # bf16 weights of an fp32 norm
    (dict(pos_dtype=5), -2, b"pos_dtype"),
    (dict(n_axes=0), -1, b"axes"),
    (dict(n_axes=5), -1, b"axes"),
    (dict(axis_dims=(3, 20, 20, 0)), -1, b"even"),
    (dict(axis_dims=(-2, 20, 20, 0)), -1, b"even"),
    (dict(axis_dims=(26, 20, 20, 0)), -1, b"exceed"),
    (dict(theta=0.0), -1, b"theta"),
    (dict(theta=float("inf")), -1, b"theta"),
    (dict(eps=-1.0), -1, b"eps"),
    (dict(eps=float("nan")), -1, b"eps"),
    (dict(norm=2), -1, b"norm"),
    (dict(q_stride=255), -1, b"strides"),
    (dict(k_stride=127), -1, b"strides"),
    (dict(pos_dtype=4), -1, b"grid"),
    (dict(pos_dtype=4, grid=(2, 3, 5)), -1, b"grid"),
    (dict(pos_dtype=4, grid=(2, 3, 4), n_axes=2), -1, b"grid"),
])
def test_rope_descriptors(kw, code, needle):
    assert rope_fwd(rope_desc(**kw)) == code
    assert needle in _lib.load().msd_last_error()


def test_rope_pointers_and_workspace():
    lib = _lib.load()
    assert rope_fwd(None) == -1 and b"NULL" in lib.msd_last_error()
    assert rope_fwd(rope_desc(), (None, 16, 16, 16, 16, 16, 16)) == -1
    assert rope_fwd(rope_desc(), (16, None, 16, 16, 16, 16, 16)) == -1
    assert rope_fwd(rope_desc(), (16, 18, 16, 16, 16, 16, 16)) == -3
    assert rope_fwd(rope_desc(), (16, 16, 18, 16, 16, 16, 16)) == -3
    assert rope_fwd(rope_desc(pos_dtype=1), (16, 16, 16, 16, 20, 16, 16)) == -3
    assert rope_fwd(rope_desc(), (16, 16, None, None, None, 16, 16)) == -1
    assert rope_fwd(rope_desc(tokens=0, pos_rows=0), (None,) * 7) == 0
    d = rope_desc()
    need = lib.msd_qk_rope_bwd_workspace_size(ctypes.byref(d))
    assert need >= 2 * 64 * 4
    assert lib.msd_qk_rope_bwd(ctypes.byref(d), *([16] * 11), 16, need - 1, None) == -4
    big = rope_desc(tokens=1 << 24, pos_rows=1 << 24)
    assert lib.msd_qk_rope_bwd_workspace_size(ctypes.byref(big)) <= 1 << 20
    plain = rope_desc(norm=0)
    assert lib.msd_qk_rope_bwd_workspace_size(ctypes.byref(plain)) == 0
    assert lib.msd_qk_rope_bwd_workspace_size(None) == 0


def test_rope_keyless_and_empty_calls():
    """A gradient of a weight that no key has is refused; no tokens need no grid."""
    lib = _lib.load()
    d = rope_desc(k_heads=0)
    assert lib.msd_qk_rope_bwd(ctypes.byref(d), *([16] * 11), 16, 1 << 30, None) == -1
    assert b"dk_weight" in lib.msd_last_error()
    assert rope_fwd(rope_desc(tokens=0, pos_rows=0, pos_dtype=4), (None,) * 7) == 0


def test_attention_sequence_limit():
    """More sequences than a launch has workgroups for are refused, as many as fit are not."""
    lib = _lib.load()
    at = attn_desc(num_seqs=1 << 20, total_q=0)
    assert attn_fwd(at, q=None, out=None) == 0
    assert attn_fwd(attn_desc(num_seqs=(1 << 20) + 1, total_q=0)) == -1
    assert b"range" in lib.msd_last_error()


def attn_desc(**kw):
    d = dict(total_q=24, total_k=40, q_stride=256, k_stride=128, v_stride=128, num_seqs=2,
             num_heads=4, num_kv_heads=2, head_dim=64, dtype=1, causal=1, scale=0.125)
    d.update(kw)
    return _lib.AttnDesc(**d)


def attn_fwd(desc, q=16, k=16, v=16, cu=16, cu_k=16, out=16, rest=None, lse=16, ws=16,
             n=1 << 40):
    return _lib.load().msd_attn_fwd(None if desc is None else ctypes.byref(desc), q, k, v, cu, cu_k,
                                    out, rest, lse, ws, n, None)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(num_heads=0), -1, b"num_heads"),
    (dict(num_kv_heads=0), -1, b"num_kv_heads"),
    (dict(num_kv_heads=3), -1, b"multiple"),
    (dict(head_dim=0), -2, b"head_dim"),
    (dict(head_dim=129, q_stride=1000, k_stride=1000, v_stride=1000), -2, b"head_dim"),
    (dict(dtype=2), -2, b"dtype"),
    (dict(causal=2), -1, b"causal"),
    (dict(num_seqs=0), -1, b"num_seqs"),
    (dict(num_seqs=1 << 30), -1, b"range"),
    (dict(total_q=-1), -1, b"range"),
    (dict(total_q=1 << 29), -1, b"range"),
    (dict(total_k=1 << 30), -1, b"range"),
    (dict(scale=0.0), -1, b"scale"),
    (dict(scale=float("nan")), -1, b"scale"),
    (dict(scale=float("inf")), -1, b"scale"),
    (dict(q_stride=255), -1, b"strides"),
    (dict(k_stride=127), -1, b"strides"),
    (dict(v_stride=0), -1, b"strides"),
])
def test_attention_descriptors(kw, code, needle):
    lib = _lib.load()
    d = attn_desc(**kw)
    assert attn_fwd(d) == code
    assert needle in lib.msd_last_error()
    assert lib.msd_attn_bwd(ctypes.byref(d), *([16] * 14), 1 << 40, None) == code
    assert lib.msd_attn_fwd_workspace_size(ctypes.byref(d)) == 0
    assert lib.msd_attn_bwd_workspace_size(ctypes.byref(d)) == 0


def test_attention_pointers_and_workspace():
    lib = _lib.load()
    assert attn_fwd(None) == -1
    assert attn_fwd(attn_desc(), q=None) == -1 and b"NULL" in lib.msd_last_error()
    assert attn_fwd(attn_desc(), k=17) == -3
    assert attn_fwd(attn_desc(), lse=18) == -3
    assert attn_fwd(attn_desc(), rest=17) == -1
    assert attn_fwd(attn_desc(dtype=0), rest=16) == -1 and b"bf16" in lib.msd_last_error()
    assert attn_fwd(attn_desc(), cu=None) == -1 and b"together" in lib.msd_last_error()
    assert attn_fwd(attn_desc(), cu_k=18) == -3
    assert attn_fwd(attn_desc(total_q=25), cu=None, cu_k=None) == -1
    assert b"multiples" in lib.msd_last_error()
    assert attn_fwd(attn_desc(total_q=0), q=None, out=None) == 0
    # one token each over long caches: the keys are split, the parts need a workspace
    d = attn_desc(num_seqs=2, total_q=2, total_k=20000)
    need = lib.msd_attn_fwd_workspace_size(ctypes.byref(d))
    assert need > 0
    assert attn_fwd(d, n=need - 1) == -4 and b"workspace" in lib.msd_last_error()
    assert attn_fwd(d, ws=None) == -4
    assert attn_fwd(d, ws=24) == -4
    d = attn_desc()
    need = lib.msd_attn_bwd_workspace_size(ctypes.byref(d))
    assert need >= 24 * 4 * 8
    assert lib.msd_attn_bwd(ctypes.byref(d), *([16] * 14), need - 1, None) == -4


def test_video_axes_and_positions():
    from megaslide_amd import video_axes, video_positions
    for hd in range(2, 257):
        ax = video_axes(hd)
        assert all(d >= 0 and d % 2 == 0 for d in ax) and hd - 1 <= sum(ax) <= hd
    p = video_positions((2, 3, 4))
    assert p.dtype == torch.int32
    n = torch.arange(24)
    assert torch.equal(p, torch.stack([n // 12, n // 4 % 3, n % 4], 1).int())


def test_no_cpu_implementation():
    from megaslide_amd import axial_rope, packed_attention, qk_norm_rope
    x = torch.zeros(6, 64)
    with pytest.raises(RuntimeError, match="ROCm"):
        axial_rope(x, (1, 2, 3), 1)
    with pytest.raises(RuntimeError, match="ROCm"):
        qk_norm_rope(x, x, None, None, (1, 2, 3), 1)
    with pytest.raises(RuntimeError, match="ROCm"):
        packed_attention(x, x, x, 1)
