// Norm of each head of q and k and rotation by the token's position on several axes, in one
// pass, forward and backward.
//
// Forward, per head row x of head_dim channels (R: the rotation, w: the norm's weight):
//   r = 1 / sqrt(mean(x^2) + eps),  y = R (w x r)          (norm = 0: y = R x)
// Pair i of axis a (even width d_a) turns by pos_a * theta^(-2 i / d_a); channels behind the
// axes pass through.  Backward, with g = R^T dy:
//   dw = sum over rows of g x r,  dx = r (w g) - x r^3 mean(w g x)   (norm = 0: dx = R^T dy)
//
// Bound: memory.  x is read and y written once (backward: x, dy read, dx written).  A workgroup
// takes a few tokens; it computes their cos and sin once into LDS (angles in revolutions, in
// 64 bits, reduced to one turn before the 32-bit functions: positions of 10^6 lose nothing) and
// then streams every head of q and of k past them, a row of 8-channel chunks per lane group,
// 16 bytes a lane.  The partner of a channel is in the lane's own chunk (interleaved pairs) or
// read through LDS (pairs half an axis apart, which no fixed shuffle serves for odd splits).
#include "common.h"
#include "qk_rope.h"

namespace msd {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTok = 8;     // tokens whose angles a workgroup holds at a time
constexpr int kMaxPairs = 128;
constexpr int kBwdBlocks = 1024;  // the weight gradient keeps one partial row per workgroup

struct RopeArgs {
  const void* x[2];        // q, k: rows of heads * hd channels, `stride` apart
  const void* w[2];        // norm weights or null
  const void* dy[2];       // backward: gradients of the results, contiguous
  void* y[2];              // forward: results, backward: gradients of x; contiguous
  int64_t stride[2];
  int heads[2];
  const void* pos;
  int64_t tokens, pos_rows;
  float* dw;               // [blocks][2][hd] partial sums of the weights' gradients, or null
  int hd, n_axes, npairs, interleaved, pos_dtype, w_f32;
  int axis[4];
  int grid[3];
  float eps;
  int tok;                 // tokens of a workgroup's step
  double rev[kMaxPairs];   // revolutions per unit of position of each pair
};

// Position of row `row` on axis x.
__device__ __forceinline__ double position(const RopeArgs& a, int64_t row, int x) {
  if (a.pos_dtype == MSD_POS_GRID) {
    const int64_t frame = static_cast<int64_t>(a.grid[1]) * a.grid[2];
    const int64_t n = x == 0 ? row / frame : row % frame;
    return static_cast<double>(x == 0 ? n : x == 1 ? n / a.grid[2] : n % a.grid[2]);
  }
  const int64_t i = row * a.n_axes + x;
  switch (a.pos_dtype) {
    case MSD_POS_I32: return static_cast<double>(static_cast<const int32_t*>(a.pos)[i]);
    case MSD_POS_I64: return static_cast<double>(static_cast<const int64_t*>(a.pos)[i]);
    case MSD_POS_F32: return static_cast<double>(static_cast<const float*>(a.pos)[i]);
    default: return static_cast<const double*>(a.pos)[i];
  }
}

// Eight channels from c0 of a row; those at or past hd read as zero.  VEC: 16-byte loads, hd a
// multiple of 8.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int c0, int hd, float (&v)[8]) {
  if (VEC) {
    if (c0 < hd) {
      if (sizeof(T) == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(p + c0);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = __uint_as_float(w[i] << 16);
          v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      } else {
        const float4 lo = *reinterpret_cast<const float4*>(p + c0);
        const float4 hi = *reinterpret_cast<const float4*>(p + c0 + 4);
        v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
        v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < hd ? to_f32(p[c0 + i]) : 0.0f;
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int c0, int hd, const float (&v)[8]) {
  if (VEC) {
    if (c0 >= hd) return;
    if (sizeof(T) == 2) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = static_cast<uint32_t>(from_f32<bf16>(v[2 * i]).bits) |
               (static_cast<uint32_t>(from_f32<bf16>(v[2 * i + 1]).bits) << 16);
      *reinterpret_cast<uint4*>(p + c0) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<float4*>(p + c0) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + c0 + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < hd) p[c0 + i] = from_f32<T>(v[i]);
  }
}

// LPR: lanes of a row (8 channels each).
template <typename T, int LPR, bool NORM, bool BWD, bool VEC>
__global__ __launch_bounds__(kThreads) void qk_rope_kernel(const RopeArgs a) {
  constexpr int kGroups = kThreads / LPR;
  __shared__ float2 s_cs[kMaxTok][kMaxPairs + 1];
  __shared__ __attribute__((aligned(16))) float s_row[kThreads * 8];
  __shared__ float s_red[BWD && NORM ? kThreads * 8 : 1];
  const int tid = threadIdx.x, lane = tid % LPR, grp = tid / LPR;
  const int c0 = lane * 8, hd = a.hd;

  // partner channel and pair of each of this lane's channels; pass-through: pair npairs
  // (cos 1, sin 0) and itself
  int other[8], pair[8];
  float sign[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = c0 + e;
    other[e] = c;
    pair[e] = a.npairs;
    sign[e] = 0.0f;
    int at = 0;
    for (int x = 0; x < a.n_axes; ++x) {
      const int d = a.axis[x], l = c - at;
      if (l >= 0 && l < d) {
        const int half = d / 2;
        const bool second = a.interleaved ? (l & 1) : l >= half;
        other[e] = a.interleaved ? (c ^ 1) : (second ? c - half : c + half);
        // axes are even and begin at even channels, so c ^ 1 is within the axis
        pair[e] = at / 2 + (a.interleaved ? l / 2 : (second ? l - half : l));
        sign[e] = second ? 1.0f : -1.0f;
      }
      at += d;
    }
    if (BWD) sign[e] = -sign[e];
  }

  float w[2][8], dw[2][8];
  if (NORM) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (a.w[t] != nullptr) {
        if (a.w_f32)
          load8<float, false>(static_cast<const float*>(a.w[t]), c0, hd, w[t]);
        else
          load8<T, false>(static_cast<const T*>(a.w[t]), c0, hd, w[t]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[t][e] = 1.0f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) dw[t][e] = 0.0f;
    }
  }

  float* const row = s_row + grp * LPR * 8;
  const int nheads = a.heads[0] + a.heads[1];
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tok; t0 < a.tokens;
       t0 += static_cast<int64_t>(gridDim.x) * a.tok) {
    const int nt = static_cast<int>(a.tokens - t0 < a.tok ? a.tokens - t0 : a.tok);
    __syncthreads();
    for (int i = tid; i < nt * (a.npairs + 1); i += kThreads) {
      const int t = i / (a.npairs + 1), p = i - t * (a.npairs + 1);
      float2 cs = make_float2(1.0f, 0.0f);
      if (p < a.npairs) {
        int x = 0, end = a.axis[0] / 2;
        while (p >= end) end += a.axis[++x] / 2;
        const double r = position(a, (t0 + t) % a.pos_rows, x) * a.rev[p];
        sincospif(2.0f * static_cast<float>(r - rint(r)), &cs.y, &cs.x);
      }
      s_cs[t][p] = cs;
    }
    __syncthreads();
    const int tasks = nt * nheads;
    for (int task = grp; task < (tasks + kGroups - 1) / kGroups * kGroups; task += kGroups) {
      const bool live = task < tasks;
      const int t = live ? task / nheads : 0, hh = live ? task - t * nheads : 0;
      const int which = hh >= a.heads[0];
      const int h = which ? hh - a.heads[0] : hh;
      const int64_t tok = t0 + t;
      const int64_t out_at = (tok * a.heads[which] + h) * hd;
      const T* xp = static_cast<const T*>(a.x[which]) + tok * a.stride[which] + int64_t(h) * hd;
      float v[8], x[8], r = 1.0f;
      if (live && (NORM || !BWD)) {
        load8<T, VEC>(xp, c0, hd, x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.0f;
      }
      if (BWD) {
        if (live) {
          load8<T, VEC>(static_cast<const T*>(a.dy[which]) + out_at, c0, hd, v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        }
      }
      if (NORM) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
        ss = group_sum<LPR>(ss);
        r = 1.0f / sqrtf(ss / hd + a.eps);
      }
      if (!BWD) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = NORM ? x[e] * r * (which ? w[1][e] : w[0][e]) : x[e];
      }
      float o[8];
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = v[e ^ 1];
      } else {
        // a row belongs to lanes of one wave: its writes and reads are in order
        *reinterpret_cast<float4*>(row + c0) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(row + c0 + 4) = make_float4(v[4], v[5], v[6], v[7]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = row[other[e]];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      float g[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 cs = s_cs[t][pair[e]];
        // a pass-through channel is not multiplied by its partner's zero (it may be infinite)
        g[e] = sign[e] == 0.0f ? v[e] : v[e] * cs.x + sign[e] * (o[e] * cs.y);
      }
      if (BWD && NORM) {
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float gx = g[e] * x[e];
          const float we = which ? w[1][e] : w[0][e];
          if (which) dw[1][e] += gx * r; else dw[0][e] += gx * r;
          dot += gx * we;
        }
        dot = group_sum<LPR>(dot);
        const float f = r * r * (r * (dot / hd));
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = r * (g[e] * (which ? w[1][e] : w[0][e])) - x[e] * f;
      }
      if (live) store8<T, VEC>(static_cast<T*>(a.y[which]) + out_at, c0, hd, g);
    }
  }

  if (BWD && NORM && a.dw != nullptr) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) s_red[grp * LPR * 8 + c0 + e] = dw[t][e];
      __syncthreads();
      for (int c = tid; c < hd; c += kThreads) {
        float s = 0.0f;
        for (int g = 0; g < kGroups; ++g) s += s_red[g * LPR * 8 + c];
        a.dw[(static_cast<int64_t>(blockIdx.x) * 2 + t) * hd + c] = s;
      }
    }
  }
}

// Sum of the workgroups' partial weight gradients, in a fixed order: 16 columns a workgroup,
// 16 threads a column.
template <typename T>
__global__ __launch_bounds__(256) void dw_sum_kernel(const float* __restrict__ part, int blocks,
                                                     int hd, T* dwq, T* dwk) {
  __shared__ float red[16][17];
  const int col = blockIdx.x * 16 + threadIdx.x % 16, r0 = threadIdx.x / 16;
  float s = 0.0f;
  if (col < 2 * hd)
    for (int b = r0; b < blocks; b += 16) s += part[static_cast<int64_t>(b) * 2 * hd + col];
  red[r0][threadIdx.x % 16] = s;
  __syncthreads();
  if (r0 == 0 && col < 2 * hd) {
    s = 0.0f;
    for (int i = 0; i < 16; ++i) s += red[i][threadIdx.x];
    T* const out = col < hd ? dwq : dwk;
    if (out != nullptr) out[col < hd ? col : col - hd] = from_f32<T>(s);
  }
}

int64_t blocks_of(const msd_qk_rope_desc& d, int tok, bool bwd) {
  const int64_t n = (d.tokens + tok - 1) / tok;
  const int64_t cap = bwd ? kBwdBlocks : int64_t(1) << 20;
  return n < cap ? n : cap;
}

// Tokens of a workgroup's step: as many as share their angles' cost, fewer where that would
// leave compute units idle (256 of them, a few workgroups each).
int tokens_of_step(const msd_qk_rope_desc& d) {
  int tok = kMaxTok;
  while (tok > 1 && d.tokens < int64_t(tok) * 1024) tok /= 2;
  return tok;
}

template <typename T, int LPR, bool NORM, bool BWD>
void launch_vec(const RopeArgs& a, unsigned blocks, bool vec, hipStream_t s) {
  if (vec)
    qk_rope_kernel<T, LPR, NORM, BWD, true><<<blocks, kThreads, 0, s>>>(a);
  else
    qk_rope_kernel<T, LPR, NORM, BWD, false><<<blocks, kThreads, 0, s>>>(a);
}

template <typename T, int LPR>
void launch_kind(const RopeArgs& a, unsigned blocks, bool norm, bool bwd, bool vec,
                 hipStream_t s) {
  if (norm && bwd) launch_vec<T, LPR, true, true>(a, blocks, vec, s);
  else if (norm) launch_vec<T, LPR, true, false>(a, blocks, vec, s);
  else if (bwd) launch_vec<T, LPR, false, true>(a, blocks, vec, s);
  else launch_vec<T, LPR, false, false>(a, blocks, vec, s);
}

template <typename T>
void launch_type(const RopeArgs& a, unsigned blocks, bool norm, bool bwd, bool vec,
                 hipStream_t s) {
  if (a.hd <= 32) launch_kind<T, 4>(a, blocks, norm, bwd, vec, s);
  else if (a.hd <= 64) launch_kind<T, 8>(a, blocks, norm, bwd, vec, s);
  else if (a.hd <= 128) launch_kind<T, 16>(a, blocks, norm, bwd, vec, s);
  else launch_kind<T, 32>(a, blocks, norm, bwd, vec, s);
}

}  // namespace

size_t qk_rope_bwd_ws_bytes(const msd_qk_rope_desc& d) {
  if (!d.norm) return 0;
  return static_cast<size_t>(blocks_of(d, tokens_of_step(d), true)) * 2 * d.head_dim * sizeof(float);
}

hipError_t launch_qk_rope(const msd_qk_rope_desc& d, const QkRopePtrs& p, bool bwd, void* ws,
                          hipStream_t s) {
  RopeArgs a{};
  for (int t = 0; t < 2; ++t) {
    a.x[t] = p.x[t];
    a.w[t] = p.w[t];
    a.dy[t] = p.dy[t];
    a.y[t] = p.y[t];
  }
  a.stride[0] = d.q_stride;
  a.stride[1] = d.k_stride;
  a.heads[0] = d.q_heads;
  a.heads[1] = d.k_heads;
  a.pos = p.pos;
  a.tokens = d.tokens;
  a.pos_rows = d.pos_rows;
  a.dw = static_cast<float*>(ws);
  a.hd = d.head_dim;
  a.n_axes = d.n_axes;
  a.interleaved = d.interleaved;
  a.pos_dtype = d.pos_dtype;
  a.w_f32 = d.weight_dtype == MSD_F32;
  a.eps = d.eps;
  for (int x = 0; x < 3; ++x) a.grid[x] = d.grid[x];
  a.tok = tokens_of_step(d);
  for (int x = 0; x < d.n_axes; ++x) {
    a.axis[x] = d.axis_dims[x];
    for (int i = 0; i < d.axis_dims[x] / 2; ++i)
      a.rev[a.npairs++] = std::pow(d.theta, -2.0 * i / d.axis_dims[x]) / 6.283185307179586476925;
  }
  const size_t e = d.dtype == MSD_BF16 ? 2 : 4;
  bool vec = d.head_dim % 8 == 0;
  for (int t = 0; t < 2; ++t) {
    if (a.heads[t] == 0) continue;
    vec = vec && (a.stride[t] * e) % 16 == 0;
    for (const void* ptr : {a.x[t], a.dy[t], static_cast<const void*>(a.y[t])})
      vec = vec && reinterpret_cast<uintptr_t>(ptr) % 16 == 0;
  }
  const unsigned blocks = static_cast<unsigned>(blocks_of(d, a.tok, bwd));
  if (blocks > 0 && d.dtype == MSD_BF16)
    launch_type<bf16>(a, blocks, d.norm != 0, bwd, vec, s);
  else if (blocks > 0)
    launch_type<float>(a, blocks, d.norm != 0, bwd, vec, s);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || !bwd || !d.norm) return err;
  const unsigned cols = static_cast<unsigned>((2 * d.head_dim + 15) / 16);
  if (a.w_f32)
    dw_sum_kernel<float><<<cols, 256, 0, s>>>(a.dw, blocks, d.head_dim,
                                              static_cast<float*>(p.dw[0]),
                                              static_cast<float*>(p.dw[1]));
  else
    dw_sum_kernel<bf16><<<cols, 256, 0, s>>>(a.dw, blocks, d.head_dim, static_cast<bf16*>(p.dw[0]),
                                             static_cast<bf16*>(p.dw[1]));
  return hipGetLastError();
}

}  // namespace msd
