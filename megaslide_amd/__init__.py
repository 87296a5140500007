"""megaslide_amd: MI355X (gfx950) HIP implementation of 3D Deformable Slide Attention.

Public surface:
  DeformableSlideAttention3D   drop-in for infinity/video/attention.py:19-273
  DenseAttention3D             dense attention with rotary (time, height, width) positions
  DiTBlock, MLP                drop-ins for infinity/video/model.py:21-117 around them
  dsa3d_core                   fused attention core (autograd; the custom
                               operator torch.ops.megaslide.dsa3d_core)
  axial_rope                   rotary positions with several axes (autograd)
  qk_norm_rope                 norm of queries and keys per head with that rotation (autograd)
  packed_attention             attention over packed sequences, grouped heads (autograd; the
                               custom operator torch.ops.megaslide.packed_attention)
  video_axes, video_positions  a head's channels per axis, a video grid's positions
  dwconv3d                     depthwise 3-D conv (+GELU) on channel-last tokens (autograd)
  keep_core_policy, keep_core_context, checkpoint_keep_core
                               selective checkpointing that keeps the core's outputs
  keep_gemms_policy, keep_gemms_context, checkpoint_keep_gemms
                               ... and every GEMM's outputs
"""

from .attention import DeformableSlideAttention3D, DenseAttention3D
from .block import MLP, DiTBlock, checkpoint_keep_core, checkpoint_keep_gemms
from .dense_ops import (axial_rope, packed_attention, qk_norm_rope, video_axes,
                        video_positions)
from .ops import (DwConv3dFunction, dsa3d_core, dwconv3d, keep_core_context, keep_core_policy,
                  keep_gemms_context, keep_gemms_policy)

__all__ = ["DeformableSlideAttention3D", "DenseAttention3D", "DiTBlock", "MLP",
           "DwConv3dFunction", "axial_rope", "dsa3d_core", "dwconv3d", "packed_attention",
           "qk_norm_rope", "video_axes", "video_positions", "keep_core_policy",
           "keep_core_context", "checkpoint_keep_core", "keep_gemms_policy",
           "keep_gemms_context", "checkpoint_keep_gemms"]
