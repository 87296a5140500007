// Attention over packed sequences, backward, in two kernels without atomics (results repeat bit
// for bit):
//
//   attn_bwd_dq_kernel   rows of queries stay, keys pass:  delta = sum(dO O) - dlse,
//                        P = exp2(c s - lse log2 e), dS = P (dO V^T - delta), dQ = scale dS K
//   attn_bwd_dkv_kernel  keys stay, the group's rows of queries pass:
//                        dV = P^T dO, dK = scale dS^T Q
//
// Seven products instead of the five that one kernel would need: recomputing S and dO V^T once
// more costs less than adding dQ up in memory, where every tile of keys would add its part of
// every row with fp32 atomics.  The stationary operands are fragments in registers, the passing
// ones tiles in LDS that are read by rows for the products over channels and by columns for
// those over rows.
#include "attn_common.h"

namespace msd {
namespace {

constexpr int kNW = 4;
constexpr int kNT = kNW * 64;
constexpr int kTile = kNW * 32;  // stationary rows of a workgroup
constexpr int kBN = 64;          // keys of a passing tile (dQ)
constexpr int kBQ = 64;          // rows of a passing tile (dK, dV)

template <typename T, int HD, bool VEC>
__global__ __launch_bounds__(kNT, 1) void attn_bwd_dq_kernel(
    const AttnArgs a, const T* __restrict__ out, const T* __restrict__ dout,
    const float* __restrict__ lse, const float* __restrict__ dlse, T* __restrict__ dq,
    float2* __restrict__ stats, int64_t slots) {
  typedef typename Elem<T>::frag Frag;
  constexpr int kKK = HD / 16, kBlk = HD / 32;
  __shared__ __attribute__((aligned(16))) T s_k[2][kBN * HD];
  __shared__ __attribute__((aligned(16))) T s_v[sizeof(T) == 2 ? 2 : 1][kBN * HD];

  int64_t id = blockIdx.x;
  const int kvh = static_cast<int>(id % a.hk);
  id /= a.hk;
  const Span sp = find_span(a, a.cu_q == nullptr ? id : slots - 1 - id, a.group, kTile, false);
  if (sp.tile < 0) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5;
  const int rows = sp.lq * a.group, shift = sp.lk - sp.lq;
  const int row0 = sp.tile * kTile + wave * 32;
  const bool mine = row0 + (lane & 31) < rows;
  const int row = mine ? row0 + (lane & 31) : rows - 1;
  const int tok = row / a.group, head = kvh * a.group + row % a.group;
  int limit = sp.lk, low = sp.lk, top = sp.lk, end = sp.lk;
  if (a.causal) {
    const int last = (sp.tile + 1) * kTile < rows ? (sp.tile + 1) * kTile : rows;
    const int wlast = row0 + 32 < rows ? row0 + 32 : rows;
    limit = tok + 1 + shift;
    low = (row0 < rows ? row0 : rows - 1) / a.group + 1 + shift;
    top = (wlast - 1) / a.group + 1 + shift;
    end = (last - 1) / a.group + 1 + shift;
    end = end > 0 ? end : 0;
  }

  const int64_t at_row = (sp.q0 + tok) * a.hq + head;
  const T* qp = static_cast<const T*>(a.q) + (sp.q0 + tok) * a.qs + int64_t(head) * a.hd;
  const T* op = out + at_row * a.hd;
  const T* gp = dout + at_row * a.hd;
  Frag q[kKK], go[kKK];
  float delta = 0.0f;
#pragma unroll
  for (int i = 0; i < kKK; ++i) {
    q[i] = mem_frag<T, VEC>(qp, i * 16 + g * 8, a.hd);
    go[i] = mem_frag<T, VEC>(gp, i * 16 + g * 8, a.hd);
    const Frag o = mem_frag<T, VEC>(op, i * 16 + g * 8, a.hd);
#pragma unroll
    for (int j = 0; j < 8; ++j) delta += static_cast<float>(go[i][j]) * static_cast<float>(o[j]);
  }
  delta = half_sum(delta);
  if (dlse != nullptr) delta -= dlse[at_row];
  float ls = lse[at_row];
  ls = ls == -INFINITY ? INFINITY : ls * kLog2e;  // a row without keys has no weights
  if (mine && g == 0) stats[at_row] = make_float2(ls, delta);

  f32x16 acc[kBlk];
#pragma unroll
  for (int b = 0; b < kBlk; ++b) acc[b] = f32x16{};
  const float c = a.scale * kLog2e;

  const int stop = (end + kBN - 1) / kBN;
  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.ks + int64_t(kvh) * a.hd;
  const T* vp = static_cast<const T*>(a.v) + sp.k0 * a.vs + int64_t(kvh) * a.hd;
  constexpr bool kTwo = sizeof(T) == 2;  // V double-buffered too (fp32: LDS holds three tiles)
  Tile<T, HD, kBN, kNT, VEC> tk, tv;
  const auto load = [&](int t) {
    const int n = sp.lk - t * kBN;
    const T* kt = kp + static_cast<int64_t>(t) * kBN * a.ks;
    const T* vt = vp + static_cast<int64_t>(t) * kBN * a.vs;
    tk.load([&](int r) { return kt + r * a.ks; }, n, a.hd);
    tv.load([&](int r) { return vt + r * a.vs; }, n, a.hd);
  };
  if (stop > 0) {
    load(0);
    tk.store(s_k[0]);
    tv.store(s_v[0]);
  }
  __syncthreads();

  for (int t = 0; t < stop; ++t) {
    const int buf = t & 1, vbuf = kTwo ? buf : 0, k0 = t * kBN;
    const bool more = t + 1 < stop;
    if (more) load(t + 1);
    if (row0 < rows && k0 < top) {
#pragma unroll
      for (int b = 0; b < kBN / 32; ++b) {
        const int kb = k0 + b * 32;
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int i = 0; i < kKK; ++i) {
          s = mma(row_frag<T, HD>(s_k[buf], b * 32 + (lane & 31), i * 16 + g * 8), q[i], s);
          dp = mma(row_frag<T, HD>(s_v[vbuf], b * 32 + (lane & 31), i * 16 + g * 8), go[i], dp);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[r] = __builtin_amdgcn_exp2f(s[r] * c - ls) * (dp[r] - delta);
        const bool masked = kb + 32 > low;
        bool bad = false;
        if (masked) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (kb + 8 * (r / 4) + 4 * g + r % 4 >= limit) s[r] = 0.0f;
          if (a.causal) {
            // keys that are not finite make the weights of rows that see them NaN; the others
            // must not meet them
#pragma unroll
            for (int d = 0; d < kBlk; ++d)
              bad |= nonfinite(col_frag<T, HD>(s_k[buf], b * 32, d)) ||
                     nonfinite(col_frag<T, HD>(s_k[buf], b * 32 + 16, d));
            bad = __any(bad);
          }
        }
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
          const Frag ds = to_frag<T>(s, t2);
#pragma unroll
          for (int d = 0; d < kBlk; ++d) {
            Frag kf = col_frag<T, HD>(s_k[buf], b * 32 + t2 * 16, d);
            if (bad) kf = finite_part(kf);
            acc[d] = mma(kf, ds, acc[d]);
          }
        }
      }
    }
    if (!kTwo) __syncthreads();
    if (more) {
      tk.store(s_k[buf ^ 1]);
      tv.store(s_v[kTwo ? buf ^ 1 : 0]);
    }
    __syncthreads();
  }
  if (!mine) return;
#pragma unroll
  for (int d = 0; d < kBlk; ++d) store_block<T, VEC>(dq + at_row * a.hd, acc[d], d, a.scale, a.hd);
}

template <typename T, int HD, bool VEC>
__global__ __launch_bounds__(kNT, 1) void attn_bwd_dkv_kernel(
    const AttnArgs a, const T* __restrict__ dout, const float2* __restrict__ stats,
    T* __restrict__ dk, T* __restrict__ dv, int64_t slots) {
  typedef typename Elem<T>::frag Frag;
  constexpr int kKK = HD / 16, kBlk = HD / 32;
  constexpr int kBufs = sizeof(T) == 2 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) T s_q[kBufs][kBQ * HD];
  __shared__ __attribute__((aligned(16))) T s_g[kBufs][kBQ * HD];
  __shared__ __attribute__((aligned(16))) float s_lse[kBufs][kBQ];
  __shared__ __attribute__((aligned(16))) float s_delta[kBufs][kBQ];

  int64_t id = blockIdx.x;
  const int kvh = static_cast<int>(id % a.hk);
  id /= a.hk;
  const Span sp = find_span(a, a.cu_k == nullptr ? id : slots - 1 - id, 1, kTile, true);
  if (sp.tile < 0) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5;
  const int rows = sp.lq * a.group, shift = sp.lk - sp.lq;
  const int key0 = sp.tile * kTile + wave * 32;
  const bool mine = key0 + (lane & 31) < sp.lk;
  const int key = mine ? key0 + (lane & 31) : sp.lk - 1;
  const int wlast = key0 + 31 < sp.lk ? key0 + 31 : sp.lk - 1;  // the wave's last key
  // rows from `first` on see this lane's key, from `wfirst` on some key of the wave, from
  // `wall` on all of them
  int first = 0, wfirst = 0, wall = 0, begin = 0;
  if (a.causal) {
    const auto from = [&](int k) {
      const int64_t i = static_cast<int64_t>(k) - shift;
      return i <= 0 ? 0 : i >= sp.lq ? rows : static_cast<int>(i) * a.group;
    };
    first = from(key);
    wfirst = from(key0 < sp.lk ? key0 : sp.lk - 1);
    wall = from(wlast);
    begin = from(sp.tile * kTile);
  }

  const T* kp = static_cast<const T*>(a.k) + (sp.k0 + key) * a.ks + int64_t(kvh) * a.hd;
  const T* vp = static_cast<const T*>(a.v) + (sp.k0 + key) * a.vs + int64_t(kvh) * a.hd;
  Frag kf[kKK], vf[kKK];
#pragma unroll
  for (int i = 0; i < kKK; ++i) {
    kf[i] = mem_frag<T, VEC>(kp, i * 16 + g * 8, a.hd);
    vf[i] = mem_frag<T, VEC>(vp, i * 16 + g * 8, a.hd);
  }
  f32x16 ak[kBlk], av[kBlk];
#pragma unroll
  for (int b = 0; b < kBlk; ++b) ak[b] = av[b] = f32x16{};
  const float c = a.scale * kLog2e;

  Tile<T, HD, kBQ, kNT, VEC> tq, tg;
  float2 st;
  const T* qbase = static_cast<const T*>(a.q) + sp.q0 * a.qs;
  const auto load = [&](int t) {
    const int r0 = t * kBQ, n = rows - r0;
    tq.load([&](int r) {
      const unsigned x = r0 + r, tok = x / static_cast<unsigned>(a.group);
      return qbase + tok * a.qs + int64_t(kvh * a.group + (x - tok * a.group)) * a.hd;
    }, n, a.hd);
    tg.load([&](int r) {
      const unsigned x = r0 + r, tok = x / static_cast<unsigned>(a.group);
      return dout + ((sp.q0 + tok) * a.hq + kvh * a.group + (x - tok * a.group)) * a.hd;
    }, n, a.hd);
    st = make_float2(INFINITY, 0.0f);
    if (tid < kBQ && tid < n) {
      const unsigned x = r0 + tid, tok = x / static_cast<unsigned>(a.group);
      st = stats[(sp.q0 + tok) * a.hq + kvh * a.group + (x - tok * a.group)];
    }
  };
  const auto store = [&](int buf) {
    tq.store(s_q[buf]);
    tg.store(s_g[buf]);
    if (tid < kBQ) {
      s_lse[buf][tid] = st.x;
      s_delta[buf][tid] = st.y;
    }
  };
  const int t0 = begin / kBQ, stop = (rows + kBQ - 1) / kBQ;
  if (t0 < stop) {
    load(t0);
    store(0);
  }
  __syncthreads();

  for (int t = t0; t < stop; ++t) {
    const int buf = kBufs == 2 ? (t - t0) & 1 : 0;
    const bool more = t + 1 < stop;
    if (more) load(t + 1);
    if (key0 < sp.lk) {
#pragma unroll
      for (int b = 0; b < kBQ / 32; ++b) {
        const int r0 = t * kBQ + b * 32;
        if (r0 + 32 <= wfirst || r0 >= rows) continue;
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int i = 0; i < kKK; ++i) {
          s = mma(row_frag<T, HD>(s_q[buf], b * 32 + (lane & 31), i * 16 + g * 8), kf[i], s);
          dp = mma(row_frag<T, HD>(s_g[buf], b * 32 + (lane & 31), i * 16 + g * 8), vf[i], dp);
        }
        f32x16 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(&s_lse[buf][b * 32 + 8 * i + 4 * g]);
          const f32x4 de = *reinterpret_cast<const f32x4*>(&s_delta[buf][b * 32 + 8 * i + 4 * g]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = 4 * i + j;
            p[r] = __builtin_amdgcn_exp2f(s[r] * c - ls[j]);
            s[r] = p[r] * (dp[r] - de[j]);
          }
        }
        const auto seen = [&](int r) { return r0 + 8 * (r / 4) + 4 * g + r % 4 >= first; };
        bool bad = false;
        if (r0 < wall) {  // causal only
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!seen(r)) p[r] = s[r] = 0.0f;
#pragma unroll
          for (int d = 0; d < kBlk; ++d)
            bad |= nonfinite(col_frag<T, HD>(s_q[buf], b * 32, d)) ||
                   nonfinite(col_frag<T, HD>(s_q[buf], b * 32 + 16, d)) ||
                   nonfinite(col_frag<T, HD>(s_g[buf], b * 32, d)) ||
                   nonfinite(col_frag<T, HD>(s_g[buf], b * 32 + 16, d));
          bad = __any(bad);
        }
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
          const Frag pf = to_frag<T>(p, t2), df = to_frag<T>(s, t2);
#pragma unroll
          for (int d = 0; d < kBlk; ++d) {
            Frag gf = col_frag<T, HD>(s_g[buf], b * 32 + t2 * 16, d);
            Frag qf = col_frag<T, HD>(s_q[buf], b * 32 + t2 * 16, d);
            if (bad) {
              gf = finite_part(gf);
              qf = finite_part(qf);
            }
            av[d] = mma(gf, pf, av[d]);
            ak[d] = mma(qf, df, ak[d]);
          }
        }
        if (bad) {
#pragma unroll
          for (int d = 0; d < kBlk; ++d)
            add_nonfinite<T>(av[d], p, seen, [&](int t2) {
              return col_frag<T, HD>(s_g[buf], b * 32 + t2 * 16, d);
            });
        }
      }
    }
    if (kBufs == 1) __syncthreads();
    if (more) store(kBufs == 2 ? buf ^ 1 : 0);
    __syncthreads();
  }
  if (!mine) return;
  const int64_t at_row = ((sp.k0 + key) * a.hk + kvh) * a.hd;
#pragma unroll
  for (int d = 0; d < kBlk; ++d) {
    store_block<T, VEC>(dk + at_row, ak[d], d, a.scale, a.hd);
    store_block<T, VEC>(dv + at_row, av[d], d, 1.0f, a.hd);
  }
}

int64_t slots_of(int64_t total, int seqs, int64_t mul, bool packed) {
  if (packed) return total * mul / kTile + seqs + 1;
  return (total / seqs * mul + kTile - 1) / kTile * seqs;
}

template <typename T, int HD, bool VEC>
hipError_t launch_hd(const AttnArgs& a, const AttnBwdPtrs& p, float2* stats, hipStream_t s) {
  const bool packed = a.cu_q != nullptr;
  const T* dout = static_cast<const T*>(p.dout);
  int64_t slots = slots_of(a.total_q, a.seqs, a.group, packed);
  if (a.total_q > 0 && slots > 0)
    attn_bwd_dq_kernel<T, HD, VEC><<<static_cast<unsigned>(slots * a.hk), kNT, 0, s>>>(
        a, static_cast<const T*>(p.out), dout, p.lse, p.dlse, static_cast<T*>(p.dq), stats, slots);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  slots = slots_of(a.total_k, a.seqs, 1, packed);
  if (a.total_k > 0 && slots > 0)
    attn_bwd_dkv_kernel<T, HD, VEC><<<static_cast<unsigned>(slots * a.hk), kNT, 0, s>>>(
        a, dout, stats, static_cast<T*>(p.dk), static_cast<T*>(p.dv), slots);
  return hipGetLastError();
}

template <typename T, int HD>
hipError_t launch_vec(const AttnArgs& a, const AttnBwdPtrs& p, float2* st, bool vec,
                      hipStream_t s) {
  return vec ? launch_hd<T, HD, true>(a, p, st, s) : launch_hd<T, HD, false>(a, p, st, s);
}

template <typename T>
hipError_t launch_type(const AttnArgs& a, const AttnBwdPtrs& p, float2* st, bool vec,
                       hipStream_t s) {
  if (a.hd <= 32) return launch_vec<T, 32>(a, p, st, vec, s);
  if (a.hd <= 64) return launch_vec<T, 64>(a, p, st, vec, s);
  if (a.hd <= 96) return launch_vec<T, 96>(a, p, st, vec, s);
  return launch_vec<T, 128>(a, p, st, vec, s);
}

}  // namespace

size_t attn_bwd_ws_bytes(const msd_attn_desc& d) {
  return static_cast<size_t>(d.total_q) * d.num_heads * sizeof(float2);
}

hipError_t launch_attn_bwd(const msd_attn_desc& d, const AttnArgs& a, const AttnBwdPtrs& p,
                           void* ws, hipStream_t s) {
  bool vec = attn_rows_aligned(a, d.dtype);
  for (const void* ptr : {p.out, p.dout, static_cast<const void*>(p.dq),
                          static_cast<const void*>(p.dk), static_cast<const void*>(p.dv)})
    vec = vec && reinterpret_cast<uintptr_t>(ptr) % 16 == 0;
  float2* const st = static_cast<float2*>(ws);
  return d.dtype == MSD_BF16 ? launch_type<bf16>(a, p, st, vec, s)
                             : launch_type<float>(a, p, st, vec, s);
}

}  // namespace msd
