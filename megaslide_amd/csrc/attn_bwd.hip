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
//
// Bound: products run in 46 to 52 % of a SIMD's cycles and vector instructions issue in 30 to 47 %;
// two waves of 250 registers a SIMD do not fill the rest, waits for LDS and, at head size 128, for a
// barrier each 32 rows.  dO V^T begins its sum with -delta, which spares a subtraction a weight (954
// -> 934 us below).
// Measured, dQ and dK/dV: 8,192 tokens, 16 x 64, bf16: 455 and 535 us, 910 and 1,030 TFLOP/s of the
// three and four products done; packed causal sequences of 129 to 5,003 tokens, 16/4 x 128: 355 and
// 480 us, 870 and 860; two fp32 clips of 2,048, 4 x 64: 130 and 154 us, 100 and 110.
#include "attn_common.h"

namespace msd {
namespace {

constexpr int kNW = 4;
constexpr int kNT = kNW * 64;
constexpr int kTile = kNW * 32;  // stationary rows of a workgroup
constexpr int kBN = 64;          // keys of a passing tile (dQ)
// dK, dV of wide bf16 heads: two accumulators of 32 keys leave no registers for the keys' and the
// values' fragments beside them at two waves a SIMD.  The values then stay in LDS, and the
// passing tiles have 32 rows instead of 64, so that two workgroups still fit a compute unit.
template <typename T, int HD>
constexpr bool kWideOf = sizeof(T) == 2 && HD > 64;
template <typename T, int HD>
constexpr int kRowsOf = kWideOf<T, HD> ? 32 : 64;  // rows of a passing tile (dK, dV)

template <typename T, int HD, bool VEC>
__global__ __launch_bounds__(kNT, sizeof(T) == 2 ? 2 : 1) void attn_bwd_dq_kernel(
    const AttnArgs a, const T* __restrict__ out, const T* __restrict__ rest,
    const T* __restrict__ dout, const float* __restrict__ lse, const float* __restrict__ dlse,
    T* __restrict__ dq, float2* __restrict__ stats, float* __restrict__ part, int nsplit) {
  typedef typename Elem<T>::frag Frag;
  constexpr int kKK = HD / 16, kBlk = HD / 32;
  __shared__ __attribute__((aligned(16))) T s_k[2][kBN * HD];
  __shared__ __attribute__((aligned(16))) T s_v[sizeof(T) == 2 ? 2 : 1][kBN * HD];

  const int hs = blockIdx.x / static_cast<unsigned>(a.hk);
  const int kvh = blockIdx.x - hs * a.hk;
  const int id = hs / nsplit, split = hs - id * nsplit;
  const Span sp = find_span(a, id, a.group, kTile, false);
  if (sp.tile < 0) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5;
  const int rows = sp.lq * a.group, shift = sp.lk - sp.lq;
  const int row0 = sp.tile * kTile + wave * 32;
  const bool mine = row0 + (lane & 31) < rows;
  const int row = mine ? row0 + (lane & 31) : rows - 1;
  const int tok = row / a.group, head = kvh * a.group + row % a.group;
  int limit = sp.lk, all = sp.lk, top = sp.lk, end = sp.lk;
  if (a.causal) {
    const int last = (sp.tile + 1) * kTile < rows ? (sp.tile + 1) * kTile : rows;
    const int wlast = row0 + 32 < rows ? row0 + 32 : rows;
    limit = tok + 1 + shift;
    all = sp.tile * kTile / a.group + 1 + shift;
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
    if (sizeof(T) == 2 && rest != nullptr) {
      const Frag x = mem_frag<T, VEC>(rest + at_row * a.hd, i * 16 + g * 8, a.hd);
#pragma unroll
      for (int j = 0; j < 8; ++j) delta += static_cast<float>(go[i][j]) * static_cast<float>(x[j]);
    }
  }
  delta = half_sum(delta);
  if (dlse != nullptr) delta -= dlse[at_row];
  float ls = lse[at_row];
  ls = ls == -INFINITY ? INFINITY : ls * kLog2e;  // a row without keys has no weights
  if (mine && g == 0 && split == 0) stats[at_row] = make_float2(ls, -delta);
  f32x16 minus;  // dO V^T - delta: the sum begins with it
#pragma unroll
  for (int r = 0; r < 16; ++r) minus[r] = -delta;

  f32x16 acc[kBlk];
#pragma unroll
  for (int b = 0; b < kBlk; ++b) acc[b] = f32x16{};
  const float c = a.scale * kLog2e;

  int first, stop;
  split_range((end + kBN - 1) / kBN, nsplit, split, &first, &stop);
  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.ks + int64_t(kvh) * a.hd;
  const T* vp = static_cast<const T*>(a.v) + sp.k0 * a.vs + int64_t(kvh) * a.hd;
  constexpr bool kTwo = sizeof(T) == 2;  // V double-buffered too (fp32: LDS holds three tiles)
  constexpr bool kDma = VEC && kTwo;
  std::conditional_t<kDma, TileDma<T, HD, kBN, kNT>, Tile<T, HD, kBN, kNT, VEC>> tk, tv;
  if constexpr (kDma) {
    tk.init(a.hd, [&](int r) { return r * a.ks; });
    tv.init(a.hd, [&](int r) { return r * a.vs; });
  }
  const auto load = [&](int t, int buf) __attribute__((always_inline)) {
    const int n = sp.lk - t * kBN;
    const T* kt = kp + static_cast<int64_t>(t) * kBN * a.ks;
    const T* vt = vp + static_cast<int64_t>(t) * kBN * a.vs;
    if constexpr (kDma) {
      tk.issue(kt, n * a.ks * 2, s_k[buf]);
      tv.issue(vt, n * a.vs * 2, s_v[buf]);
    } else {
      tk.load([&](int r, int) { return kt + r * a.ks; }, n, a.hd);
      tv.load([&](int r, int) { return vt + r * a.vs; }, n, a.hd);
    }
  };
  const auto arrive = [&](int buf) __attribute__((always_inline)) {
    if constexpr (kDma) {
      dma_wait();
    } else {
      tk.store(s_k[buf]);
      tv.store(s_v[kTwo ? buf : 0]);
    }
  };
  if (first < stop) {
    load(first, 0);
    arrive(0);
  }
  __syncthreads();

  Finite<T> fin;
  const auto step = [&](int t, auto masked_c) __attribute__((always_inline)) {
    constexpr bool kMasked = decltype(masked_c)::value;
    const int buf = (t - first) & 1, vbuf = kTwo ? buf : 0, k0 = t * kBN;
    const bool more = t + 1 < stop;
    if (more) load(t + 1, buf ^ 1);
    if (row0 < rows && (!kMasked || k0 < top)) {
#pragma unroll
      for (int b = 0; b < kBN / 32; ++b) {
        f32x16 s = {}, dp = minus;
#pragma unroll
        for (int i = 0; i < kKK; ++i) {
          s = mma(row_frag<T, HD>(s_k[buf], b * 32 + (lane & 31), i * 16 + g * 8), q[i], s);
          dp = mma(row_frag<T, HD>(s_v[vbuf], b * 32 + (lane & 31), i * 16 + g * 8), go[i], dp);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = __builtin_amdgcn_exp2f(s[r] * c - ls) * dp[r];
          if (kMasked && k0 + b * 32 + 8 * (r / 4) + 4 * g + r % 4 >= limit) s[r] = 0.0f;
        }
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
          const Frag ds = to_frag<T>(s, t2);
#pragma unroll
          for (int d = 0; d < kBlk; ++d) {
            Frag kf = col_frag<T, HD>(s_k[buf], b * 32 + t2 * 16, d);
            // (a row that sees a key that is not finite has weights that are NaN)
            if (kMasked) kf = fin(kf);
            acc[d] = mma(kf, ds, acc[d]);
          }
        }
      }
    }
    if (!kTwo) __syncthreads();
    if (more) arrive(buf ^ 1);
    __syncthreads();
  };
  int t = first, whole = all > 0 ? all / kBN : 0;  // tiles that every row sees whole
  whole = whole < stop ? whole : stop;
  for (; t < whole; ++t) step(t, std::false_type{});
  for (; t < stop; ++t) step(t, std::true_type{});
  if (!mine) return;
  float* const po = part + (split * a.total_q * a.hq + at_row) * HD;
#pragma unroll
  for (int d = 0; d < kBlk; ++d) {
    if (nsplit > 1)
      store_block<float, true>(po, acc[d], d, a.scale, HD);
    else
      store_block<T, VEC>(dq + at_row * a.hd, acc[d], d, a.scale, a.hd);
  }
}

template <typename T, int HD, bool VEC>
__global__ __launch_bounds__(kNT, sizeof(T) == 2 ? 2 : 1) void attn_bwd_dkv_kernel(
    const AttnArgs a, const T* __restrict__ dout, const float2* __restrict__ stats,
    T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part, int nsplit) {
  typedef typename Elem<T>::frag Frag;
  constexpr int kKK = HD / 16, kBlk = HD / 32;
  constexpr int kBufs = sizeof(T) == 2 ? 2 : 1, kBQ = kRowsOf<T, HD>;
  constexpr bool kWide = kWideOf<T, HD>;
  // the tiles that loads fill directly come first: such loads reach 64 KB of LDS
  __shared__ struct {
    alignas(16) T q[kBufs][kBQ * HD];
    alignas(16) T g[kBufs][kBQ * HD];
    alignas(16) T v[kWide ? kTile * HD : 8];
    alignas(16) float lse[kBufs][kBQ];
    alignas(16) float delta[kBufs][kBQ];
  } sm;
  auto& s_q = sm.q;
  auto& s_g = sm.g;
  auto& s_v = sm.v;
  auto& s_lse = sm.lse;
  auto& s_delta = sm.delta;

  const int hs = blockIdx.x / static_cast<unsigned>(a.hk);
  const int kvh = blockIdx.x - hs * a.hk;
  const int id = hs / nsplit, split = hs - id * nsplit;
  const Span sp = find_span(a, id, 1, kTile, true);
  if (sp.tile < 0) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5;
  const int rows = sp.lq * a.group, shift = sp.lk - sp.lq;
  const int key0 = sp.tile * kTile + wave * 32;
  const bool mine = key0 + (lane & 31) < sp.lk;
  const int key = mine ? key0 + (lane & 31) : sp.lk - 1;
  // rows from `first` on see this lane's key, from `wfirst` on some key of the wave, from
  // `begin` on some key of the workgroup, from `all` on all of them
  int first = 0, wfirst = 0, all = 0, begin = 0;
  if (a.causal) {
    const auto from = [&](int k) {
      const int64_t i = static_cast<int64_t>(k) - shift;
      return i <= 0 ? 0 : i >= sp.lq ? rows : static_cast<int>(i) * a.group;
    };
    first = from(key);
    wfirst = from(key0 < sp.lk ? key0 : sp.lk - 1);
    const int last = (sp.tile + 1) * kTile - 1;
    all = from(last < sp.lk ? last : sp.lk - 1);
    begin = from(sp.tile * kTile);
  }

  const T* kp = static_cast<const T*>(a.k) + (sp.k0 + key) * a.ks + int64_t(kvh) * a.hd;
  const T* vp = static_cast<const T*>(a.v) + (sp.k0 + key) * a.vs + int64_t(kvh) * a.hd;
  Frag kf[kKK], vf[kWide ? 1 : kKK];
#pragma unroll
  for (int i = 0; i < kKK; ++i) {
    kf[i] = mem_frag<T, VEC>(kp, i * 16 + g * 8, a.hd);
    const Frag v = mem_frag<T, VEC>(vp, i * 16 + g * 8, a.hd);
    if constexpr (kWide)  // in the order in which this very lane reads it: one address for all
      *reinterpret_cast<Frag*>(s_v + ((wave * kKK + i) * 64 + lane) * 8) = v;
    else
      vf[i] = v;
  }
  f32x16 ak[kBlk], av[kBlk];
#pragma unroll
  for (int b = 0; b < kBlk; ++b) ak[b] = av[b] = f32x16{};
  const float c = a.scale * kLog2e;

  // A tile has as many whole tokens of the group's heads as its rows hold, so that every tile is
  // laid out alike; groups of more than 32 heads (not VEC) divide for every row.
  const int toks = VEC ? kBQ / a.group : 0, trows = VEC ? toks * a.group : kBQ;
  constexpr bool kDma = VEC && sizeof(T) == 2;
  std::conditional_t<kDma, TileDma<T, HD, kBQ, kNT>, Tile<T, HD, kBQ, kNT, VEC>> tq, tg;
  const int64_t gs = static_cast<int64_t>(a.hq) * a.hd;
  const T* qbase = static_cast<const T*>(a.q) + sp.q0 * a.qs + int64_t(kvh) * a.group * a.hd;
  const T* gbase = dout + sp.q0 * gs + int64_t(kvh) * a.group * a.hd;
  const float2* sbase = stats + sp.q0 * a.hq + kvh * a.group;
  const auto row_off = [&](int r, int64_t stride) -> int64_t {
    if (r >= trows) return -1;
    const int tok = r / a.group;
    return tok * stride + (r - tok * a.group) * a.hd;
  };
  const int64_t soff = tid < kBQ ? (tid < trows ? tid / a.group * static_cast<int64_t>(a.hq) +
                                                      tid % a.group
                                                : 0)
                                 : 0;
  int64_t qoff[kDma || !VEC ? 1 : decltype(tq)::kItems], goff[kDma || !VEC ? 1 : decltype(tq)::kItems];
  if constexpr (kDma) {
    tq.init(a.hd, [&](int r) { return row_off(r, a.qs); });
    tg.init(a.hd, [&](int r) { return row_off(r, gs); });
  } else if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < decltype(tq)::kItems; ++i) {
      const int r = (tid + i * kNT) / decltype(tq)::kChunks;
      qoff[i] = row_off(r, a.qs);
      goff[i] = row_off(r, gs);
    }
  }
  float2 st;
  const auto load = [&](int t, int buf) __attribute__((always_inline)) {
    const int r0 = t * trows;
    const int n = rows - r0 < trows ? rows - r0 : trows;
    st = make_float2(INFINITY, 0.0f);
    if constexpr (VEC) {
      const int64_t tok0 = static_cast<int64_t>(t) * toks;
      const T* qt = qbase + tok0 * a.qs;
      const T* gt = gbase + tok0 * gs;
      if constexpr (kDma) {
        const int64_t left = sp.lq - tok0;
        tq.issue(qt, left * a.qs * 2, s_q[buf]);
        tg.issue(gt, left * gs * 2, s_g[buf]);
      } else {
        tq.load([&](int, int i) { return qt + qoff[i]; }, n, a.hd);
        tg.load([&](int, int i) { return gt + goff[i]; }, n, a.hd);
      }
      if (tid < n) st = sbase[tok0 * a.hq + soff];
    } else {
      const auto at = [&](int r, int64_t stride) {
        const unsigned x = r0 + r, tok = x / static_cast<unsigned>(a.group);
        return tok * stride + static_cast<int64_t>(x - tok * a.group) * a.hd;
      };
      tq.load([&](int r, int) { return qbase + at(r, a.qs); }, n, a.hd);
      tg.load([&](int r, int) { return gbase + at(r, gs); }, n, a.hd);
      if (tid < n) {
        const unsigned x = r0 + tid, tok = x / static_cast<unsigned>(a.group);
        st = sbase[static_cast<int64_t>(tok) * a.hq + (x - tok * a.group)];
      }
    }
  };
  const auto arrive = [&](int buf) __attribute__((always_inline)) {
    if (tid < kBQ) {
      s_lse[buf][tid] = st.x;
      s_delta[buf][tid] = st.y;
    }
    if constexpr (kDma) {
      dma_wait();
    } else {
      tq.store(s_q[buf]);
      tg.store(s_g[buf]);
    }
  };
  int t0, stop;
  split_range((rows + trows - 1) / trows - begin / trows, nsplit, split, &t0, &stop);
  t0 += begin / trows;
  stop += begin / trows;
  if (t0 < stop) {
    load(t0, 0);
    arrive(0);
  }
  __syncthreads();

  Finite<T> finq, fing;
  const auto step = [&](int t, auto masked_c) __attribute__((always_inline)) {
    constexpr bool kMasked = decltype(masked_c)::value;
    const int buf = kBufs == 2 ? (t - t0) & 1 : 0;
    const bool more = t + 1 < stop;
    if (more) load(t + 1, kBufs == 2 ? buf ^ 1 : 0);
    if (key0 < sp.lk) {
#pragma unroll
      for (int b = 0; b < kBQ / 32; ++b) {
        const int r0 = t * trows + b * 32;
        if (kMasked && r0 + 32 <= wfirst) continue;
        f32x16 s = {}, dp;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 de = *reinterpret_cast<const f32x4*>(&s_delta[buf][b * 32 + 8 * i + 4 * g]);
#pragma unroll
          for (int j = 0; j < 4; ++j) dp[4 * i + j] = de[j];
        }
#pragma unroll
        for (int i = 0; i < kKK; ++i) {
          s = mma(row_frag<T, HD>(s_q[buf], b * 32 + (lane & 31), i * 16 + g * 8), kf[i], s);
          Frag v;
          if constexpr (kWide)
            v = *reinterpret_cast<const Frag*>(s_v + ((wave * kKK + i) * 64 + lane) * 8);
          else
            v = vf[i];
          dp = mma(row_frag<T, HD>(s_g[buf], b * 32 + (lane & 31), i * 16 + g * 8), v, dp);
        }
        f32x16 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(&s_lse[buf][b * 32 + 8 * i + 4 * g]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = 4 * i + j;
            p[r] = __builtin_amdgcn_exp2f(s[r] * c - ls[j]);
            s[r] = p[r] * dp[r];
            if (kMasked && r0 + 8 * i + 4 * g + j < first) p[r] = s[r] = 0.0f;
          }
        }
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
          const Frag pf = to_frag<T>(p, t2), df = to_frag<T>(s, t2);
#pragma unroll
          for (int d = 0; d < kBlk; ++d) {
            Frag gf = col_frag<T, HD>(s_g[buf], b * 32 + t2 * 16, d);
            Frag qf = col_frag<T, HD>(s_q[buf], b * 32 + t2 * 16, d);
            if (kMasked) {
              gf = fing(gf);
              qf = finq(qf);  // (a query that is not finite makes the weights it has NaN)
            }
            av[d] = mma(gf, pf, av[d]);
            ak[d] = mma(qf, df, ak[d]);
          }
        }
      }
    }
    if (kBufs == 1) __syncthreads();
    if (more) arrive(kBufs == 2 ? buf ^ 1 : 0);
    __syncthreads();
  };
  int t = t0, cut = (all + trows - 1) / trows;  // tiles from `cut` on see every key
  cut = cut < t0 ? t0 : cut < stop ? cut : stop;
  for (; t < cut; ++t) step(t, std::true_type{});
  for (; t < stop; ++t) step(t, std::false_type{});
  if (__any(fing.bad()))
    add_nonfinite<T>(
        av, t0 * trows, cut * trows < rows ? cut * trows : rows, a.hd,
        [=](int r) {
          const int tok = r / a.group;
          return gbase + tok * gs + static_cast<int64_t>(r - tok * a.group) * a.hd;
        },
        [=](int r) { return r >= first; });
  if (!mine) return;
  const int64_t at_row = (sp.k0 + key) * a.hk + kvh, n = a.total_k * a.hk;
  float* const po = part + (split * n + at_row) * HD;
#pragma unroll
  for (int d = 0; d < kBlk; ++d) {
    if (nsplit > 1) {
      store_block<float, true>(po, ak[d], d, a.scale, HD);
      store_block<float, true>(po + nsplit * n * HD, av[d], d, 1.0f, HD);
    } else {
      store_block<T, VEC>(dk + at_row * a.hd, ak[d], d, a.scale, a.hd);
      store_block<T, VEC>(dv + at_row * a.hd, av[d], d, 1.0f, a.hd);
    }
  }
}

// Adds the parts of gradients whose sums were split, in order: rows of HD floats to rows of hd
// values; blockIdx.y: which of two (dk, dv).
template <typename T>
__global__ __launch_bounds__(256) void attn_add_kernel(const float* __restrict__ part, int nsplit,
                                                       int64_t rows, int hd, int padded, T* out0,
                                                       T* out1) {
  const int quads = padded / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = i / quads;
  const int c = static_cast<int>(i - row * quads) * 4;
  if (row >= rows || c >= hd) return;
  const float* p = part + (blockIdx.y * nsplit * rows + row) * padded + c;
  f32x4 s = *reinterpret_cast<const f32x4*>(p);
  for (int k = 1; k < nsplit; ++k) s += *reinterpret_cast<const f32x4*>(p + k * rows * padded);
  T* const o = (blockIdx.y ? out1 : out0) + row * hd + c;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j < hd) o[j] = from_f32<T>(s[j]);
}

int64_t slots_of(int64_t total, int seqs, int64_t mul, bool packed) {
  if (packed) return total * mul / kTile + seqs + 1;
  return (total / seqs * mul + kTile - 1) / kTile * seqs;
}

// Workgroups along the other side's rows where the tiles alone leave compute units idle, or end
// late with the longest sequence's tiles: `wgs` workgroups, a mean of `passing` tiles to pass.
// (Two fp32 clips of 2,048 tokens, 4 heads x 64, 140 workgroups: 276 us in two parts, 296 in four,
// 330 in eight.  bf16, 420 workgroups of sequences of 129 to 5,003 tokens: dK/dV 1,250 us whole,
// 950 in three parts.)
int splits(int64_t wgs, int64_t passing, int dtype) {
  const int64_t enough = dtype == MSD_BF16 ? 1024 : 256;
  if (wgs == 0 || wgs >= (dtype == MSD_BF16 ? 512 : 256)) return 1;
  int64_t n = (enough + wgs - 1) / wgs;
  const int64_t most = (passing + 3) / 4;  // four tiles each at least
  n = n < most ? n : most;
  return static_cast<int>(n < 1 ? 1 : n > 16 ? 16 : n);
}

struct Plan {
  int64_t q_slots, k_slots;
  int q_split, k_split;
};

Plan plan(const msd_attn_desc& d, bool packed) {
  const int group = d.num_heads / d.num_kv_heads;
  Plan p;
  p.q_slots = d.total_q > 0 ? slots_of(d.total_q, d.num_seqs, group, packed) : 0;
  p.k_slots = d.total_k > 0 ? slots_of(d.total_k, d.num_seqs, 1, packed) : 0;
  const int64_t keys = d.total_k / d.num_seqs / kBN, rows = d.total_q / d.num_seqs * group / 64;
  p.q_split = splits(p.q_slots * d.num_kv_heads, keys, d.dtype);
  p.k_split = splits(p.k_slots * d.num_kv_heads, rows, d.dtype);
  return p;
}

int padded_hd(int hd) { return (hd + 31) / 32 * 32; }

size_t part_bytes(const msd_attn_desc& d, bool packed) {
  const Plan p = plan(d, packed);
  const int64_t q = p.q_split > 1 ? p.q_split * d.total_q * d.num_heads : 0;
  const int64_t k = p.k_split > 1 ? 2 * p.k_split * d.total_k * d.num_kv_heads : 0;
  return static_cast<size_t>(q > k ? q : k) * padded_hd(d.head_dim) * sizeof(float);
}

size_t stats_bytes(const msd_attn_desc& d) {
  return (static_cast<size_t>(d.total_q) * d.num_heads * sizeof(float2) + 255) / 256 * 256;
}

template <typename T, int HD, bool VEC>
hipError_t launch_hd(const msd_attn_desc& d, const AttnArgs& a, const AttnBwdPtrs& p, void* ws,
                     hipStream_t s) {
  const Plan pl = plan(d, a.cu_q != nullptr);
  const T* dout = static_cast<const T*>(p.dout);
  T* const dq = static_cast<T*>(p.dq);
  T* const dk = static_cast<T*>(p.dk);
  T* const dv = static_cast<T*>(p.dv);
  float2* const stats = static_cast<float2*>(ws);
  // dq's parts are added up before dk's and dv's take their place
  float* const part = reinterpret_cast<float*>(static_cast<char*>(ws) + stats_bytes(d));
  const auto add = [&](int n, int64_t rows, T* o0, T* o1) {
    attn_add_kernel<T><<<dim3(static_cast<unsigned>((rows * (HD / 4) + 255) / 256), o1 ? 2 : 1),
                         256, 0, s>>>(part, n, rows, a.hd, HD, o0, o1);
  };
  if (pl.q_slots > 0) {
    attn_bwd_dq_kernel<T, HD, VEC>
        <<<static_cast<unsigned>(pl.q_slots * pl.q_split * a.hk), kNT, 0, s>>>(
            a, static_cast<const T*>(p.out), static_cast<const T*>(p.rest), dout, p.lse, p.dlse, dq,
            stats, part, pl.q_split);
    if (pl.q_split > 1) add(pl.q_split, a.total_q * a.hq, dq, nullptr);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (pl.k_slots > 0) {
    attn_bwd_dkv_kernel<T, HD, VEC>
        <<<static_cast<unsigned>(pl.k_slots * pl.k_split * a.hk), kNT, 0, s>>>(
            a, dout, stats, dk, dv, part, pl.k_split);
    if (pl.k_split > 1) add(pl.k_split, a.total_k * a.hk, dk, dv);
  }
  return hipGetLastError();
}

template <typename T, int HD>
hipError_t launch_vec(const msd_attn_desc& d, const AttnArgs& a, const AttnBwdPtrs& p, void* ws,
                      bool vec, hipStream_t s) {
  return vec ? launch_hd<T, HD, true>(d, a, p, ws, s) : launch_hd<T, HD, false>(d, a, p, ws, s);
}

template <typename T>
hipError_t launch_type(const msd_attn_desc& d, const AttnArgs& a, const AttnBwdPtrs& p, void* ws,
                       bool vec, hipStream_t s) {
  switch (padded_hd(a.hd)) {
    case 32: return launch_vec<T, 32>(d, a, p, ws, vec, s);
    case 64: return launch_vec<T, 64>(d, a, p, ws, vec, s);
    case 96: return launch_vec<T, 96>(d, a, p, ws, vec, s);
    default: return launch_vec<T, 128>(d, a, p, ws, vec, s);
  }
}

}  // namespace

// Upper bound over both forms (packed or equal lengths): the descriptor does not say which.
size_t attn_bwd_ws_bytes(const msd_attn_desc& d) {
  const size_t x = part_bytes(d, true), y = part_bytes(d, false);
  return stats_bytes(d) + (x > y ? x : y);
}

hipError_t launch_attn_bwd(const msd_attn_desc& d, const AttnArgs& a, const AttnBwdPtrs& p,
                           void* ws, hipStream_t s) {
  bool vec = attn_vec(d, a, true);
  for (const void* ptr : {p.out, p.rest, p.dout, static_cast<const void*>(p.dq),
                          static_cast<const void*>(p.dk), static_cast<const void*>(p.dv)})
    vec = vec && reinterpret_cast<uintptr_t>(ptr) % 16 == 0;
  return d.dtype == MSD_BF16 ? launch_type<bf16>(d, a, p, ws, vec, s)
                             : launch_type<float>(d, a, p, ws, vec, s);
}

}  // namespace msd
