// Norm of each head of q and k and rotation by the token's position on several axes, in one
// pass, forward and backward.
//
// Forward, per head row x of head_dim channels (R: the rotation, w: the norm's weight):
//   r = 1 / sqrt(mean(x^2) + eps),  y = R (w x r)          (norm = 0: y = R x)
// Pair i of axis a (even width d_a) turns by pos_a * theta^(-2 i / d_a); channels behind the
// axes pass through.  Backward, with g = R^T dy:
//   dw = sum over rows of g x r,  dx = r (w g) - x r^3 mean(w g x)   (norm = 0: dx = R^T dy)
//
// Bound: memory.  x is read and y written once (backward: x, dy read, dx written).  A wave takes
// a token: its lanes compute the cos and sin of the token's pairs once into LDS (angles in
// revolutions, in 64 bits, reduced to one turn before the 32-bit functions: positions of 10^6
// lose nothing), each lane takes those of its 8 channels into registers, and the heads stream
// past, a row per lane group, 16 bytes a lane, the next rows (the next token's after the last)
// in flight meanwhile.  Workgroups of q and of k are apart: one tensor's weights fit the
// registers beside two rows in flight.  The partner of a channel is in
// the lane's own chunk (interleaved pairs) or read through LDS (pairs half an axis apart, which
// no fixed shuffle serves for odd splits).  Where tokens are few, their heads are split among
// workgroups.
// Measured (a copy reaches 5.1 TB/s): rotation of 46,800 tokens, 16 x 96, bf16, 65 us forward and
// 65 backward, 4.4 TB/s; with the norm, 65,536 tokens, 16 + 16 heads x 64, bf16, 130 and 180 us, 4.1
// and 4.5 TB/s; 32,768 tokens, 8 + 8 x 64, fp32, 64 and 83 us, 4.2 and 4.8 TB/s; 16 tokens 6 us.
#include "common.h"
#include "qk_rope.h"

#include <type_traits>

namespace msd {
namespace {

constexpr int kMaxPairs = 128;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
// As many workgroups as the compute units hold at a time (the norm's backward, with one partial
// row of the weights' gradients each, half as many): what a lane knows of its channels and the
// weights is then set up once for many tokens.
constexpr int kMaxBlocks = 2048;
constexpr int kMaxBwdBlocks = 1024;

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
  int hd, n_axes, npairs, pos_dtype, w_f32, pass;
  int axis[4];
  int grid[3];
  float eps;
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

// Eight channels from c0 of a row as they are stored; those at or past hd are zeros.  VEC:
// 16-byte loads, hd a multiple of 8.
template <typename T>
struct Raw {
  uint4 u[sizeof(T) / 2];

  template <bool VEC>
  __device__ __forceinline__ void load(const T* p, int c0, int hd, bool live) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) u[i] = make_uint4(0, 0, 0, 0);
    if (!live) return;
    if (VEC) {
      if (c0 < hd) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
          u[i] = reinterpret_cast<const uint4*>(p + c0)[i];
      }
    } else {
      union {
        T e[8];
        uint4 v[sizeof(T) / 2];
      } x;
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) x.v[i] = u[i];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < hd) x.e[i] = p[c0 + i];
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) u[i] = x.v[i];
    }
  }

  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (sizeof(T) == 2) {
      const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    }
  }
};

template <typename T>
__device__ __forceinline__ void load_weight(const void* p, int c0, int hd, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = c0 + i < hd ? to_f32(static_cast<const T*>(p)[c0 + i]) : 0.0f;
}

// PAST: past the caches.
template <typename T, bool VEC, bool PAST>
__device__ __forceinline__ void store8(T* p, int c0, int hd, const float (&v)[8]) {
  if (VEC) {
    if (c0 >= hd) return;
    if constexpr (sizeof(T) == 2) {
      typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
      bf16x8 r;
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = static_cast<__bf16>(v[i]);
      if constexpr (PAST)
        __builtin_nontemporal_store(r, reinterpret_cast<bf16x8*>(p + c0));
      else
        *reinterpret_cast<bf16x8*>(p + c0) = r;
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

// LDS of one wave: its writes are in order before its reads.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Sum over the LPR lanes of a row, the same bits in each; `buf`: the row's floats in LDS.
template <int LPR>
__device__ __forceinline__ float row_sum(float v, int sub, float* buf) {
  if constexpr ((LPR & (LPR - 1)) == 0) {
    return group_sum<LPR>(v);
  } else {
    buf[sub] = v;
    wave_fence();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < LPR; ++i) s += buf[i];
    wave_fence();
    return s;
  }
}

// LPR: lanes of a row (8 channels each).
template <typename T, int LPR, bool NORM, bool BWD, bool VEC, bool INTER, bool PAST = false>
__global__ __launch_bounds__(kThreads, 4) void qk_rope_kernel(const RopeArgs a) {
  constexpr int kRows = 64 / LPR;  // rows of a wave at a time (lanes behind them idle)
  constexpr int kAhead = sizeof(T) == 2 && !(NORM && BWD) ? 2 : 1;  // rows of a lane in flight
  constexpr bool kExchange = !INTER || (NORM && (LPR & (LPR - 1)) != 0);
  constexpr bool kRowBuf = kExchange || (NORM && BWD);
  __shared__ float2 s_cs[kWaves][kMaxPairs + 1];
  __shared__ __attribute__((aligned(16))) float s_row[kRowBuf ? kThreads * 8 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sub = lane % LPR, grp = lane / LPR;  // grp == kRows: an idle lane
  const int c0 = sub * 8, hd = a.hd;

  // of each of this lane's channels: its pair (pass-through: npairs, cos 1, sin 0), partner << 8
  // and, at bit 16, whether the partner's term is subtracted
  int code[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = c0 + e;
    code[e] = a.npairs | (c << 8);
    int at = 0;
    for (int x = 0; x < a.n_axes; ++x) {
      const int d = a.axis[x], l = c - at;
      // (an idle lane stays within its own slot of s_row)
      if (l >= 0 && l < d && (64 % LPR == 0 || grp < kRows)) {
        const int half = d / 2;
        // axes are even and begin at even channels, so c ^ 1 is within the axis
        const bool second = INTER ? (l & 1) : l >= half;
        const int other = INTER ? (c ^ 1) : (second ? c - half : c + half);
        const int pair = at / 2 + (INTER ? l / 2 : (second ? l - half : l));
        code[e] = pair | (other << 8) | (second == BWD ? 1 << 16 : 0);  // backward: turns back
      }
      at += d;
    }
  }

  const int which = blockIdx.z;  // 0: q, 1: k
  const int heads = a.heads[which];
  float w[8], dw[8];
  if (NORM) {
    if (a.w[which] == nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.0f;
    } else if (a.w_f32) {
      load_weight<float>(a.w[which], c0, hd, w);
    } else {
      load_weight<T>(a.w[which], c0, hd, w);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[e] = 0.0f;
  }

  float* const row = s_row + (kRowBuf ? (wave * 64 + grp * LPR) * 8 : 0);
  if (lane == 0) s_cs[wave][a.npairs] = make_float2(1.0f, 0.0f);
  const float inv_hd = 1.0f / hd;

  // heads [h0, h1) are this workgroup's
  const int per = (heads + gridDim.y - 1) / gridDim.y;
  const int h0 = blockIdx.y * per, h1 = h0 + per < heads ? h0 + per : heads;
  const T* const xs = static_cast<const T*>(a.x[which]);
  const T* const dys = static_cast<const T*>(a.dy[which]);
  T* const ys = static_cast<T*>(a.y[which]);
  const int64_t stride = a.stride[which], out_stride = static_cast<int64_t>(heads) * hd;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWaves;

  Raw<T> rx[kAhead], ry[kAhead];  // the next rows
  const auto load = [&](int64_t tok, int h) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int hh = h + i * kRows + grp;
      const bool live = hh < h1 && grp < kRows;
      if (NORM || !BWD) rx[i].template load<VEC>(xs + tok * stride + hh * hd, c0, hd, live);
      if (BWD) ry[i].template load<VEC>(dys + tok * out_stride + hh * hd, c0, hd, live);
    }
  };
  int64_t tok = static_cast<int64_t>(blockIdx.x) * kWaves + wave;
  if (tok < a.tokens) load(tok, h0);
  for (; tok < a.tokens; tok += step) {
    wave_fence();
    const int64_t prow = a.pos_rows == a.tokens ? tok : tok % a.pos_rows;
    for (int p = lane; p < a.npairs; p += 64) {
      int x = 0, end = a.axis[0] / 2;
      while (p >= end) end += a.axis[++x] / 2;
      const double r = position(a, prow, x) * a.rev[p];
      float2 cs;
      sincospif(2.0f * static_cast<float>(r - rint(r)), &cs.y, &cs.x);
      s_cs[wave][p] = cs;
    }
    wave_fence();
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 v = s_cs[wave][code[e] & 255];
      cs[e] = v.x;
      sn[e] = code[e] & (1 << 16) ? -v.y : v.y;
    }

    for (int h = h0; h < h1; h += kAhead * kRows) {
      Raw<T> cx[kAhead], cy[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        cx[i] = rx[i];
        cy[i] = ry[i];
      }
      if (h + kAhead * kRows < h1)
        load(tok, h + kAhead * kRows);
      else if (tok + step < a.tokens)
        load(tok + step, h0);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int hh = h + i * kRows + grp;
        if (h + i * kRows >= h1) break;
        float v[8], x[8], r = 1.0f;
        if (NORM || !BWD) cx[i].get(x);
        if (BWD) cy[i].get(v);
        if (NORM) {
          float ss = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
          ss = row_sum<LPR>(ss, sub, row);
          r = rsqrtf(ss * inv_hd + a.eps);
        }
        if (!BWD) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = NORM ? x[e] * r * w[e] : x[e];
        }
        float o[8];
        if (INTER) {
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = v[e ^ 1];
        } else {
          *reinterpret_cast<float4*>(row + c0) = make_float4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<float4*>(row + c0 + 4) = make_float4(v[4], v[5], v[6], v[7]);
          wave_fence();
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = row[(code[e] >> 8) & 255];
          wave_fence();
        }
        float g[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = v[e] * cs[e] + sn[e] * o[e];
        if (a.pass) {
          // channels that pass through are not multiplied by zero (they may be infinite)
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = (code[e] & 255) == a.npairs ? v[e] : g[e];
        }
        if (BWD && NORM) {
          float dot = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            dw[e] += g[e] * x[e] * r;
            g[e] *= w[e];
            dot += g[e] * x[e];
          }
          dot = row_sum<LPR>(dot, sub, row);
          const float f = r * r * (r * (dot * inv_hd));
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = r * g[e] - x[e] * f;
        }
        if (hh < h1 && grp < kRows)
          store8<T, VEC, PAST>(ys + tok * out_stride + hh * hd, c0, hd, g);
      }
    }
  }

  if (BWD && NORM && a.dw != nullptr) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) row[c0 + e] = dw[e];
    __syncthreads();
    for (int c = tid; c < hd; c += kThreads) {
      float s = 0.0f;
      for (int g = 0; g < kWaves * kRows; ++g)
        s += s_row[(g / kRows * 64 + g % kRows * LPR) * 8 + c];
      const int64_t blk = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
      a.dw[(blk * 2 + which) * hd + c] = s;
    }
  }
}

// Sum of the workgroups' partial weight gradients, in a fixed order: 16 columns a workgroup,
// 64 threads a column.
template <typename T>
__global__ __launch_bounds__(1024) void dw_sum_kernel(const float* __restrict__ part, int blocks,
                                                      int hd, T* dwq, T* dwk) {
  __shared__ float red[64][17];
  const int col = blockIdx.x * 16 + threadIdx.x % 16, r0 = threadIdx.x / 16;
  float s = 0.0f;
  if (col < 2 * hd) {
#pragma unroll 4
    for (int b = r0; b < blocks; b += 64) s += part[static_cast<int64_t>(b) * 2 * hd + col];
  }
  red[r0][threadIdx.x % 16] = s;
  __syncthreads();
  if (r0 == 0 && col < 2 * hd) {
    s = 0.0f;
    for (int i = 0; i < 64; ++i) s += red[i][threadIdx.x];
    T* const out = col < hd ? dwq : dwk;
    if (out != nullptr) out[col < hd ? col : col - hd] = from_f32<T>(s);
  }
}

// Lanes of a head's row: 10 and 12 (head sizes to 80 and 96) leave 4 of 64 lanes idle where 16
// would leave 24 and 16.
int lanes_of(int hd) {
  for (int n : {4, 8, 10, 12, 16})
    if (hd <= 8 * n) return n;
  return 32;
}

struct Shape {
  int64_t x;  // workgroups along the tokens
  int y;      // and along the heads
};

// One token a wave; where that is under 2,048 waves (eight a compute unit), the heads are split
// too, down to one row of a lane group each.
Shape grid_of(const msd_qk_rope_desc& d, bool bwd) {
  const int rows = 64 / lanes_of(d.head_dim);
  const int steps = (d.q_heads + rows - 1) / rows;
  Shape s{(d.tokens + kWaves - 1) / kWaves, 1};
  while (s.y * 2 <= steps && d.tokens * s.y < 2048) s.y *= 2;
  const int64_t cap = bwd && d.norm ? kMaxBwdBlocks : kMaxBlocks;
  if (s.x > cap) s.x = cap;
  return s;
}

template <typename T, int LPR, bool NORM, bool BWD>
void launch_vec(const RopeArgs& a, Shape g, bool vec, bool inter, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(g.x), g.y, a.heads[1] > 0 ? 2 : 1);
  // Results of more than half the 256 MB behind the L2s go past the caches, where they would not
  // stay until they are read (144 and 268 MB, forward and backward: 137 -> 133 and 310 -> 297 us; fp32,
  // 134 MB: 152 -> 157, so in bf16 only).
  if constexpr (sizeof(T) == 2) {
    const int64_t values = a.tokens * (a.heads[0] + static_cast<int64_t>(a.heads[1])) * a.hd;
    if (vec && values * 2 > (int64_t(128) << 20)) {
      if (inter)
        qk_rope_kernel<T, LPR, NORM, BWD, true, true, true><<<grid, kThreads, 0, s>>>(a);
      else
        qk_rope_kernel<T, LPR, NORM, BWD, true, false, true><<<grid, kThreads, 0, s>>>(a);
      return;
    }
  }
  if (vec && inter) qk_rope_kernel<T, LPR, NORM, BWD, true, true><<<grid, kThreads, 0, s>>>(a);
  else if (vec) qk_rope_kernel<T, LPR, NORM, BWD, true, false><<<grid, kThreads, 0, s>>>(a);
  else if (inter) qk_rope_kernel<T, LPR, NORM, BWD, false, true><<<grid, kThreads, 0, s>>>(a);
  else qk_rope_kernel<T, LPR, NORM, BWD, false, false><<<grid, kThreads, 0, s>>>(a);
}

template <typename T, int LPR>
void launch_kind(const RopeArgs& a, Shape g, bool norm, bool bwd, bool vec, bool inter,
                 hipStream_t s) {
  if (norm && bwd) launch_vec<T, LPR, true, true>(a, g, vec, inter, s);
  else if (norm) launch_vec<T, LPR, true, false>(a, g, vec, inter, s);
  else if (bwd) launch_vec<T, LPR, false, true>(a, g, vec, inter, s);
  else launch_vec<T, LPR, false, false>(a, g, vec, inter, s);
}

template <typename T>
void launch_type(const RopeArgs& a, Shape g, bool norm, bool bwd, bool vec, bool inter,
                 hipStream_t s) {
  switch (lanes_of(a.hd)) {
    case 4: return launch_kind<T, 4>(a, g, norm, bwd, vec, inter, s);
    case 8: return launch_kind<T, 8>(a, g, norm, bwd, vec, inter, s);
    case 10: return launch_kind<T, 10>(a, g, norm, bwd, vec, inter, s);
    case 12: return launch_kind<T, 12>(a, g, norm, bwd, vec, inter, s);
    case 16: return launch_kind<T, 16>(a, g, norm, bwd, vec, inter, s);
    default: return launch_kind<T, 32>(a, g, norm, bwd, vec, inter, s);
  }
}

}  // namespace

size_t qk_rope_bwd_ws_bytes(const msd_qk_rope_desc& d) {
  if (!d.norm) return 0;
  const Shape g = grid_of(d, true);
  return static_cast<size_t>(g.x) * g.y * 2 * d.head_dim * sizeof(float);
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
  a.pos_dtype = d.pos_dtype;
  a.w_f32 = d.weight_dtype == MSD_F32;
  a.eps = d.eps;
  for (int x = 0; x < 3; ++x) a.grid[x] = d.grid[x];
  for (int x = 0; x < d.n_axes; ++x) {
    // theta^(-2 i / d) by products in extended precision: a few steps of 2^-64 off
    const long double step = powl(static_cast<long double>(d.theta), -2.0L / d.axis_dims[x]);
    long double f = 1.0L / 6.283185307179586476925287L;
    a.axis[x] = d.axis_dims[x];
    for (int i = 0; i < d.axis_dims[x] / 2; ++i, f *= step) a.rev[a.npairs++] = static_cast<double>(f);
  }
  a.pass = 2 * a.npairs < d.head_dim;
  const size_t e = d.dtype == MSD_BF16 ? 2 : 4;
  bool vec = d.head_dim % 8 == 0;
  for (int t = 0; t < 2; ++t) {
    if (a.heads[t] == 0) continue;
    vec = vec && (a.stride[t] * e) % 16 == 0;
    for (const void* ptr : {a.x[t], a.dy[t], static_cast<const void*>(a.y[t])})
      vec = vec && reinterpret_cast<uintptr_t>(ptr) % 16 == 0;
  }
  const Shape g = grid_of(d, bwd);
  if (g.x > 0 && d.dtype == MSD_BF16)
    launch_type<bf16>(a, g, d.norm != 0, bwd, vec, d.interleaved != 0, s);
  else if (g.x > 0)
    launch_type<float>(a, g, d.norm != 0, bwd, vec, d.interleaved != 0, s);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || !bwd || !d.norm) return err;
  const unsigned cols = static_cast<unsigned>((2 * d.head_dim + 15) / 16);
  const int blocks = static_cast<int>(g.x * g.y);
  if (a.w_f32)
    dw_sum_kernel<float><<<cols, 1024, 0, s>>>(a.dw, blocks, d.head_dim,
                                               static_cast<float*>(p.dw[0]),
                                               static_cast<float*>(p.dw[1]));
  else
    dw_sum_kernel<bf16><<<cols, 1024, 0, s>>>(a.dw, blocks, d.head_dim,
                                              static_cast<bf16*>(p.dw[0]),
                                              static_cast<bf16*>(p.dw[1]));
  return hipGetLastError();
}

}  // namespace msd
