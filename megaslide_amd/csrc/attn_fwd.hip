// Attention over packed sequences, forward: out = softmax(scale q k^T + mask) v.
//
// Rows of a workgroup are (query token, head of the group) pairs of one key head, so a tile of
// keys and values is read once for all heads that share it; one token's heads are rows of one
// block.  One pass over the keys with the running maximum m and sum l of a softmax (fp32):
// S^T = K Q^T, p = exp2(c (s - m)), O^T += V^T P^T, each a block of the matrix cores with the
// rows along the lanes, so that m, l and the rescale of O are one value a lane and P is a
// fragment where it stands.  m is raised only where a score exceeds it by 2^8 or more in p
// (p <= 256: nothing is lost in fp32), which spares most rescales.
//
// Bound: the vector unit beside the matrix cores.  Of the cycles of a SIMD vector instructions issue
// in 73 % and products run in 45 % (8,192 tokens, 16 x 64, bf16, four waves a SIMD; 46 % and 41 % at
// 16/4 heads x 128, causal, two waves); LDS is busy for 20 %, and nine in ten requests hit the L2.  Four waves of 32 rows and 64 keys: eight waves, or 32 keys,
// were 7 to 10 % slower, and so was the forward without the search for the maximum on the small
// head sizes.  Tiles that a causal mask cuts are a loop of their own, so that the others compare
// nothing.
// Measured: 8,192 tokens, 16 x 64, bf16: 308 us, 890 TFLOP/s (a library product of that type
// 1,300 to 1,570); packed sequences of 129 to 5,003 tokens, causal, 16/4 x 128: 239 us, 870; prompts
// of 1 to 4,096, causal, 32/8 x 128: 233 us, 820; two fp32 clips of 2,048, 4 x 64: 96 us,
// 90 TFLOP/s (a library product 153).
#include "attn_common.h"

namespace msd {
namespace {

constexpr int kBN = 64;  // keys of a tile

template <typename T, int HD, int NW, bool VEC>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 ? (HD <= 64 ? 4 : 2) : 1) void attn_fwd_kernel(
    const AttnArgs a, T* __restrict__ out, T* __restrict__ rest, float* __restrict__ lse,
    float* __restrict__ part, int nsplit) {
  typedef typename Elem<T>::frag Frag;
  constexpr int kBM = NW * 32, kNT = NW * 64, kKK = HD / 16, kBlk = HD / 32, kSB = kBN / 32;
  __shared__ __attribute__((aligned(16))) T s_k[2][kBN * HD];
  __shared__ __attribute__((aligned(16))) T s_v[2][kBN * HD];

  // key head fastest: neighbours on the eight dies take different heads, and a head's tiles
  // keep to one die's L2 where the heads are a multiple of eight
  const unsigned id = blockIdx.x, hs = id / a.hk;
  const int kvh = id - hs * a.hk;
  const int slot = hs / nsplit, split = hs - slot * nsplit;
  const Span sp = find_span(a, slot, a.group, kBM, false);
  if (sp.tile < 0) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5;
  const int rows = sp.lq * a.group;  // the ABI keeps this below 2^31
  const int shift = sp.lk - sp.lq;
  const int row0 = sp.tile * kBM + wave * 32;
  const int row = row0 + (lane & 31) < rows ? row0 + (lane & 31) : rows - 1;
  const int tok = row / a.group, head = kvh * a.group + row % a.group;
  // keys before `limit` are seen by this lane's row, before `top` by some row of the wave, before
  // `all` by every row of the workgroup, before `end` by some row of it
  int limit = sp.lk, all = sp.lk, top = sp.lk, end = sp.lk;
  if (a.causal) {
    const int last = (sp.tile + 1) * kBM < rows ? (sp.tile + 1) * kBM : rows;
    const int wlast = row0 + 32 < rows ? row0 + 32 : rows;
    limit = tok + 1 + shift;
    all = sp.tile * kBM / a.group + 1 + shift;
    top = (wlast - 1) / a.group + 1 + shift;
    end = (last - 1) / a.group + 1 + shift;
    end = end > 0 ? end : 0;
  }

  const T* qp = static_cast<const T*>(a.q) + (sp.q0 + tok) * a.qs + int64_t(head) * a.hd;
  Frag q[kKK];
#pragma unroll
  for (int i = 0; i < kKK; ++i) q[i] = mem_frag<T, VEC>(qp, i * 16 + g * 8, a.hd);

  f32x16 o[kBlk];
#pragma unroll
  for (int b = 0; b < kBlk; ++b) o[b] = f32x16{};
  float m = -INFINITY, l = 0.0f;
  const float c = a.scale * kLog2e;

  int first, stop;
  split_range((end + kBN - 1) / kBN, nsplit, split, &first, &stop);
  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.ks + int64_t(kvh) * a.hd;
  const T* vp = static_cast<const T*>(a.v) + sp.k0 * a.vs + int64_t(kvh) * a.hd;
  // bf16 rows of 16-byte chunks go straight to LDS, others through registers
  constexpr bool kDma = VEC && sizeof(T) == 2;
  std::conditional_t<kDma, TileDma<T, HD, kBN, kNT>, Tile<T, HD, kBN, kNT, VEC>> tk, tv;
  if constexpr (kDma) {
    tk.init(a.hd, [&](int r) { return r * a.ks; });
    tv.init(a.hd, [&](int r) { return r * a.vs; });
  }
  // starts tile t on its way to buffer `buf`, and ends it
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
      tv.store(s_v[buf]);
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
    const int buf = (t - first) & 1, k0 = t * kBN;
    const bool more = t + 1 < stop;
    if (more) load(t + 1, buf ^ 1);
    if (row0 < rows && (!kMasked || k0 < top)) {
      f32x16 s[kSB];
#pragma unroll
      for (int b = 0; b < kSB; ++b) {
        s[b] = f32x16{};
#pragma unroll
        for (int i = 0; i < kKK; ++i)
          s[b] = mma(row_frag<T, HD>(s_k[buf], b * 32 + (lane & 31), i * 16 + g * 8), q[i], s[b]);
      }
      if (kMasked) {
#pragma unroll
        for (int b = 0; b < kSB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (k0 + b * 32 + 8 * (r / 4) + 4 * g + r % 4 >= limit) s[b][r] = -INFINITY;
      }
      float top_s = s[0][0];
#pragma unroll
      for (int b = 0; b < kSB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) top_s = fmaxf(top_s, s[b][r]);
      top_s = half_max(top_s);
      if (__any((top_s - m) * c > 8.0f)) {
        const float m_new = fmaxf(m, top_s);
        const float f = m_new == -INFINITY ? 1.0f : exp2f((m - m_new) * c);
        l *= f;
#pragma unroll
        for (int b = 0; b < kBlk; ++b) o[b] *= f;
        m = m_new;
      }
      const float mc = m == -INFINITY ? 0.0f : m * c;
#pragma unroll
      for (int b = 0; b < kSB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[b][r] = __builtin_amdgcn_exp2f(s[b][r] * c - mc);
          l += s[b][r];
        }
#pragma unroll
      for (int b = 0; b < kSB; ++b)
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
          const Frag p = to_frag<T>(s[b], t2);
#pragma unroll
          for (int d = 0; d < kBlk; ++d) {
            Frag v = col_frag<T, HD>(s_v[buf], b * 32 + t2 * 16, d);
            if (kMasked) v = fin(v);
            o[d] = mma(v, p, o[d]);
          }
        }
    }
    if (more) arrive(buf ^ 1);
    __syncthreads();
  };
  int t = first, whole = all > 0 ? all / kBN : 0;  // tiles that every row sees whole
  whole = whole < stop ? whole : stop;
  for (; t < whole; ++t) step(t, std::false_type{});
  const int cut = t;
  for (; t < stop; ++t) step(t, std::true_type{});
  if (__any(fin.bad()))
    add_nonfinite<T>(
        o, cut * kBN, stop * kBN < sp.lk ? stop * kBN : sp.lk, a.hd,
        [=](int r) { return vp + r * a.vs; }, [=](int r) { return r < limit; });

  l = half_sum(l);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const float ls = l == 0.0f ? -INFINITY : m * a.scale + logf(l);
  if (row0 + (lane & 31) >= rows) return;
  const int64_t at_row = (sp.q0 + tok) * a.hq + head;
  if (nsplit > 1) {
    const int64_t r = split * a.total_q * a.hq + at_row;
    float* po = part + r * HD;
#pragma unroll
    for (int d = 0; d < kBlk; ++d) store_block<float, true>(po, o[d], d, inv, HD);
    if (g == 0) part[static_cast<int64_t>(nsplit) * a.total_q * a.hq * HD + r] = ls;
  } else {
    T* op = out + at_row * a.hd;
#pragma unroll
    for (int d = 0; d < kBlk; ++d) store_block<T, VEC>(op, o[d], d, inv, a.hd);
    if (sizeof(T) == 2 && rest != nullptr) {
#pragma unroll
      for (int d = 0; d < kBlk; ++d)
        store_rest<T, VEC>(rest + at_row * a.hd, o[d], d, inv, a.hd);
    }
    if (lse != nullptr && g == 0) lse[at_row] = ls;
  }
}

// Joins the parts of rows whose keys were split: out = sum_i exp(lse_i - lse) out_i.  One wave
// a row.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(const float* __restrict__ part,
                                                        int nsplit, int64_t rows, int hd,
                                                        int stride, T* __restrict__ out,
                                                        T* __restrict__ rest,
                                                        float* __restrict__ lse) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 64;
  const int lane = threadIdx.x & 63;
  if (row >= rows) return;
  const float* ls = part + nsplit * rows * stride;
  float m = -INFINITY;
  for (int i = lane; i < nsplit; i += 64) m = fmaxf(m, ls[i * rows + row]);
  for (int x = 32; x > 0; x /= 2) m = fmaxf(m, __shfl_xor(m, x));
  const float base = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < nsplit; ++i) {
    const float li = ls[i * rows + row];
    if (li == -INFINITY) continue;  // no key of this row in that part
    const float w = exp2f((li - base) * kLog2e);
    sum += w;
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (lane + 64 * x < hd) acc[x] += w * part[(i * rows + row) * stride + lane + 64 * x];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (lane + 64 * x < hd) {
      out[row * hd + lane + 64 * x] = from_f32<T>(acc[x] * inv);
      if (rest != nullptr)
        rest[row * hd + lane + 64 * x] = from_f32<T>(rest_of<T>(acc[x] * inv));
    }
  if (lse != nullptr && lane == 0) lse[row] = sum == 0.0f ? -INFINITY : base + logf(sum);
}

// One new token each over caches: as many workgroups a sequence and key head as it has
// chunks of keys, so that long and short caches share the device evenly.  Bound: memory, K and V
// once.  The group's heads are the rows of one block; the NW waves take every NW-th tile of 32
// keys of the chunk for themselves and meet only at its end, so no wave waits for another.
// A wave's next keys are on their way to LDS while it weighs the present values, and the next
// values while it scores the next keys.  Parts are joined by attn_join_tokens_kernel.
// 131,000 keys of 16 sequences, 32/8 heads x 128: 112 us, 4.8 TB/s (a copy reaches 5.1), and 7
// for the join; 119 with both launches.
template <typename T, int HD>
constexpr int kTokenWaves = sizeof(T) == 4 && HD > 64 ? 2 : 4;  // their tiles fill 64 KB of LDS

template <typename T, int HD>
__global__ __launch_bounds__((kTokenWaves<T, HD> * 64), sizeof(T) == 4 ? 1 : 2)
void attn_tokens_kernel(const AttnArgs a, T* __restrict__ out, T* __restrict__ rest,
                        float* __restrict__ lse, float* __restrict__ part, int chunk,
                        int64_t units) {
  typedef typename Elem<T>::frag Frag;
  constexpr int kKK = HD / 16, kBlk = HD / 32, kN = 32, NW = kTokenWaves<T, HD>;
  constexpr int kLoads = TileDma<T, HD, kN, 64>::kItems;
  // the tiles that loads fill directly come first: such loads reach 64 KB of LDS
  __shared__ struct {
    union {
      struct {
        alignas(16) T k[kN * HD], v[kN * HD];
      } w[NW];
      float o[NW][32][HD];
    };
    float m[NW][32], l[NW][32];
  } sm;

  const int slot = blockIdx.x / static_cast<unsigned>(a.hk);
  const int kvh = blockIdx.x - slot * a.hk;
  const Span sp = find_span(a, slot, 1, chunk, true);
  if (sp.tile < 0 || sp.lq == 0) return;
  const int lane = threadIdx.x & 63, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = kvh * a.group + ((lane & 31) < a.group ? lane & 31 : 0);
  const int64_t kbase = a.cu_k == nullptr ? static_cast<int64_t>(sp.seq) * a.nk
                                          : bound_of(a.cu_k, sp.seq, a.total_k);
  const int64_t unit = kbase / chunk + sp.seq + sp.tile;
  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.ks + int64_t(kvh) * a.hd;
  const T* vp = static_cast<const T*>(a.v) + sp.k0 * a.vs + int64_t(kvh) * a.hd;
  T* const sk = sm.w[wave].k;
  T* const sv = sm.w[wave].v;
  TileDma<T, HD, kN, 64> tk, tv;
  tk.init(a.hd, [&](int r) { return r * a.ks; });
  tv.init(a.hd, [&](int r) { return r * a.vs; });
  const float c = a.scale * kLog2e;

  // A sequence's first token by chunks; further ones, which this kernel is not made for, whole,
  // by the workgroup of the first chunk.
  const int toks = sp.tile == 0 ? sp.lq : 1;
  for (int tok = 0; tok < toks; ++tok) {
    int limit = sp.lk;
    if (a.causal) {
      limit = tok + 1 + sp.lk - sp.lq;
      limit = limit < 0 ? 0 : limit;
    }
    const int from = tok == 0 ? sp.tile * chunk : 0;
    int to = tok == 0 && from + chunk < limit ? from + chunk : limit;
    to = to < from ? from : to;
    const T* qp = static_cast<const T*>(a.q) + (sp.q0 + tok) * a.qs + int64_t(head) * a.hd;
    Frag q[kKK];
#pragma unroll
    for (int i = 0; i < kKK; ++i) q[i] = mem_frag<T, true>(qp, i * 16 + g * 8, a.hd);
    f32x16 o[kBlk];
#pragma unroll
    for (int b = 0; b < kBlk; ++b) o[b] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    const auto load_k = [&](int k0) __attribute__((always_inline)) {
      tk.issue(kp + k0 * a.ks, (sp.lk - k0) * a.ks * int64_t(sizeof(T)), sk);
    };
    const auto load_v = [&](int k0) __attribute__((always_inline)) {
      tv.issue(vp + k0 * a.vs, (sp.lk - k0) * a.vs * int64_t(sizeof(T)), sv);
    };
    int64_t k0 = from + wave * kN;
    if (k0 < to) {
      load_k(k0);
      load_v(k0);
    }
    for (; k0 < to; k0 += NW * kN) {
      dma_wait<kLoads>();  // the keys
      f32x16 s = {};
#pragma unroll
      for (int i = 0; i < kKK; ++i)
        s = mma(row_frag<T, HD>(sk, lane & 31, i * 16 + g * 8), q[i], s);
      const bool more = k0 + NW * kN < to;
      // (all reads of the tile are back before it is overwritten)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) load_k(k0 + NW * kN);
      if (k0 + kN > to) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 8 * (r / 4) + 4 * g + r % 4 >= to) s[r] = -INFINITY;
      }
      float top_s = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top_s = fmaxf(top_s, s[r]);
      top_s = half_max(top_s);
      if (__any((top_s - m) * c > 8.0f)) {
        const float m_new = fmaxf(m, top_s);
        const float f = m_new == -INFINITY ? 1.0f : exp2f((m - m_new) * c);
        l *= f;
#pragma unroll
        for (int b = 0; b < kBlk; ++b) o[b] *= f;
        m = m_new;
      }
      const float mc = m == -INFINITY ? 0.0f : m * c;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(s[r] * c - mc);
        l += s[r];
      }
      if (more)
        dma_wait<kLoads>();  // the values
      else
        dma_wait();
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        const Frag p = to_frag<T>(s, t2);
#pragma unroll
        for (int d = 0; d < kBlk; ++d) {
          Frag v = col_frag<T, HD>(sv, t2 * 16, d);
          // keys behind the limit have weight zero, and their values may not be finite
          if (k0 + kN > to) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (k0 + t2 * 16 + (j / 4) * 8 + 4 * g + j % 4 >= to) v[j] = 0;
          }
          o[d] = mma(v, p, o[d]);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) load_v(k0 + NW * kN);
    }
    l = half_sum(l);

    // the waves' parts, of the group's rows
    __syncthreads();
    if ((lane & 31) < a.group) {
#pragma unroll
      for (int d = 0; d < kBlk; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4*>(&sm.o[wave][lane & 31][d * 32 + 8 * i + 4 * g]) =
              f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
      if (g == 0) {
        sm.m[wave][lane & 31] = m;
        sm.l[wave][lane & 31] = l;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.group * HD; i += NW * 64) {
      const int row = i / HD, ch = i - row * HD;
      float top = -INFINITY, acc = 0.0f, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) top = fmaxf(top, sm.m[w][row]);
      const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = exp2f((sm.m[w][row] - base) * c);
        acc += f * sm.o[w][row][ch];
        sum += f * sm.l[w][row];
      }
      const float ls = sum == 0.0f ? -INFINITY : top * a.scale + logf(sum);
      acc = sum == 0.0f ? 0.0f : acc / sum;
      if (tok == 0) {
        const int64_t r = (unit * a.hk + kvh) * a.group + row;
        part[r * HD + ch] = acc;
        if (ch == 0) part[units * a.hq * HD + r] = ls;
      } else {
        const int64_t r = (sp.q0 + tok) * a.hq + kvh * a.group + row;
        if (ch < a.hd) out[r * a.hd + ch] = from_f32<T>(acc);
        if (ch < a.hd && rest != nullptr)
          rest[r * a.hd + ch] = from_f32<T>(rest_of<T>(acc));
        if (ch == 0 && lse != nullptr) lse[r] = ls;
      }
    }
    __syncthreads();
  }
}

// Joins the chunks of every sequence's first token, one workgroup a (row, head), its waves every
// eighth chunk each; rows that no key belongs to (behind the last sequence, or of a sequence
// without keys) become 0 and -inf.  Bound: latency, of parts that other dies wrote: a wave has
// eight of them on their way at a time (256 parts of 16 rows: 19 -> 7 us against four waves that
// took them one after the other).
constexpr int kJoinWaves = 8;

template <typename T>
__global__ __launch_bounds__(kJoinWaves * 64) void attn_join_tokens_kernel(
    const AttnArgs a, const float* __restrict__ part, int chunk, int64_t units, int hd_padded,
    T* __restrict__ out, T* __restrict__ rest, float* __restrict__ lse) {
  __shared__ float s_acc[kJoinWaves][128], s_sum[kJoinWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.x / static_cast<unsigned>(a.hq);
  const int head = blockIdx.x - row * a.hq;
  int s;  // the last sequence that begins at or before the row: as many offsets are not above it
  int64_t first = row, lk = a.nk, kbase;
  if (a.cu_q == nullptr) {
    s = row;
    kbase = static_cast<int64_t>(s) * a.nk;
  } else {
    s = 0;
    for (int i = 1; i <= a.seqs; i += 64)
      s += __builtin_popcountll(
          __ballot(i + lane <= a.seqs && bound_of(a.cu_q, i + lane, a.total_q) <= row));
    first = bound_of(a.cu_q, s, a.total_q);
    kbase = bound_of(a.cu_k, s, a.total_k);
    const int64_t e = s < a.seqs ? bound_of(a.cu_k, s + 1, a.total_k) : 0;
    lk = e > kbase ? e - kbase : 0;
  }
  if (s < a.seqs && lk > 0 && row != first) return;  // written whole
  const int n = s < a.seqs ? static_cast<int>((lk + chunk - 1) / chunk) : 0;
  const int64_t unit = kbase / chunk + s;
  const float* ls = part + units * a.hq * hd_padded + unit * a.hq + head;
  const float* po = part + (unit * a.hq + head) * hd_padded;
  const int64_t step = static_cast<int64_t>(a.hq);
  float m = -INFINITY;
  for (int k = lane; k < n; k += 64) m = fmaxf(m, ls[k * step]);
  for (int x = 32; x > 0; x /= 2) m = fmaxf(m, __shfl_xor(m, x));
  const float base = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f, acc[2] = {0.0f, 0.0f};
  for (int k0 = wave; k0 < n; k0 += 8 * kJoinWaves) {
    float w[8], v[8][2];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int k = k0 + u * kJoinWaves;
      w[u] = k < n ? ls[k * step] : -INFINITY;
#pragma unroll
      for (int x = 0; x < 2; ++x)
        v[u][x] = k < n && lane + 64 * x < a.hd ? po[k * step * hd_padded + lane + 64 * x] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float f = exp2f((w[u] - base) * kLog2e);
      sum += f;
#pragma unroll
      for (int x = 0; x < 2; ++x) acc[x] += f * v[u][x];
    }
  }
  s_acc[wave][lane] = acc[0];
  s_acc[wave][lane + 64] = acc[1];
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kJoinWaves; ++w) sum += s_sum[w];
  const int ch = threadIdx.x;
  const int64_t r = static_cast<int64_t>(row) * a.hq + head;
  if (ch < a.hd) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) v += s_acc[w][ch];
    v = sum == 0.0f ? 0.0f : v / sum;
    out[r * a.hd + ch] = from_f32<T>(v);
    if (rest != nullptr) rest[r * a.hd + ch] = from_f32<T>(rest_of<T>(v));
  }
  if (lse != nullptr && ch == 0) lse[r] = sum == 0.0f ? -INFINITY : base + logf(sum);
}

int padded_hd(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 96 ? 96 : 128; }

int64_t q_slots(const msd_attn_desc& d, bool packed, int tile) {
  const int64_t group = d.num_heads / d.num_kv_heads;
  if (!packed) return d.total_q / d.num_seqs == 0 ? 0 : d.num_seqs * ((d.total_q / d.num_seqs * group + tile - 1) / tile);
  return d.total_q * group / tile + d.num_seqs + 1;
}

// Workgroups along the keys: enough that the launch fills the 256 compute units, several times in
// bf16, where two to four workgroups share one and sequences differ, each with 256 keys at least
// of a sequence of mean length.  (Two fp32 clips of 2,048 tokens, 4 heads x 64: 164 us whole, 106
// in two parts, 114 in four, 128 in eight.)
int splits(const msd_attn_desc& d, bool packed, int tile) {
  const int64_t wgs = q_slots(d, packed, tile) * d.num_kv_heads;
  const int64_t enough = d.dtype == MSD_BF16 ? 1024 : 256;
  if (wgs == 0 || wgs >= (d.dtype == MSD_BF16 ? 512 : 256)) return 1;
  const int64_t mean = d.total_k / d.num_seqs;
  int64_t n = (enough + wgs - 1) / wgs;
  const int64_t most = mean / 256;
  n = n < most ? n : most;
  return static_cast<int>(n < 1 ? 1 : n > 256 ? 256 : n);
}

constexpr int kNW = 4;

// Keys of a workgroup of attn_tokens_kernel: about 2,048 workgroups in all, 256 to 2,048 keys.
// 0: not its case.  One token a sequence is what total_q == num_seqs suggests (other lengths are
// right too, and slower); a group is the rows of one block; below 1,024 keys in all the kernel
// that needs no joining is faster.
int token_chunk(const msd_attn_desc& d) {
  if (d.total_q != d.num_seqs || d.num_heads / d.num_kv_heads > 32 || d.total_k < 1024)
    return 0;
  const int64_t n = (d.total_k * d.num_kv_heads / 2048 + 127) / 128 * 128;
  return static_cast<int>(n < 256 ? 256 : n > 2048 ? 2048 : n);
}

int64_t token_units(const msd_attn_desc& d, int chunk) {
  return d.total_k / chunk + d.num_seqs + 1;
}

template <typename T, int HD>
hipError_t launch_tokens(const msd_attn_desc& d, const AttnArgs& a, T* out, T* rest, float* lse,
                         float* ws, int chunk, hipStream_t s) {
  const int64_t units = token_units(d, chunk);
  int64_t slots = units;
  if (a.cu_q == nullptr) slots = (d.total_k / d.num_seqs + chunk - 1) / chunk * d.num_seqs;
  attn_tokens_kernel<T, HD>
      <<<static_cast<unsigned>(slots * a.hk), kTokenWaves<T, HD> * 64, 0, s>>>(
          a, out, rest, lse, ws, chunk, units);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  attn_join_tokens_kernel<T><<<static_cast<unsigned>(a.total_q * a.hq), kJoinWaves * 64, 0, s>>>(
      a, ws, chunk, units, HD, out, rest, lse);
  return hipGetLastError();
}

template <typename T, int HD>
hipError_t launch_hd(const msd_attn_desc& d, const AttnArgs& a, T* out, T* rest, float* lse,
                     float* ws, bool vec, hipStream_t s) {
  const int chunk = vec ? token_chunk(d) : 0;
  if (chunk > 0) return launch_tokens<T, HD>(d, a, out, rest, lse, ws, chunk, s);
  const bool packed = a.cu_q != nullptr;
  const int n = splits(d, packed, kNW * 32);
  const int64_t slots = q_slots(d, packed, kNW * 32);
  const int64_t blocks = slots * n * a.hk;
  if (blocks == 0) return hipSuccess;
  if (vec)
    attn_fwd_kernel<T, HD, kNW, true>
        <<<static_cast<unsigned>(blocks), kNW * 64, 0, s>>>(a, out, rest, lse, ws, n);
  else
    attn_fwd_kernel<T, HD, kNW, false>
        <<<static_cast<unsigned>(blocks), kNW * 64, 0, s>>>(a, out, rest, lse, ws, n);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || n == 1) return e;
  const int64_t rows = a.total_q * a.hq;
  attn_join_kernel<T><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, s>>>(ws, n, rows, a.hd, HD,
                                                                           out, rest, lse);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const msd_attn_desc& d, const AttnArgs& a, void* out, void* rest,
                       float* lse, void* ws, bool vec, hipStream_t s) {
  T* o = static_cast<T*>(out);
  T* r = static_cast<T*>(rest);
  float* w = static_cast<float*>(ws);
  switch (padded_hd(a.hd)) {
    case 32: return launch_hd<T, 32>(d, a, o, r, lse, w, vec, s);
    case 64: return launch_hd<T, 64>(d, a, o, r, lse, w, vec, s);
    case 96: return launch_hd<T, 96>(d, a, o, r, lse, w, vec, s);
    default: return launch_hd<T, 128>(d, a, o, r, lse, w, vec, s);
  }
}

}  // namespace

int attn_max_head_dim() { return 128; }

AttnArgs attn_args(const msd_attn_desc& d, const void* q, const void* k, const void* v,
                   const int32_t* cu_q, const int32_t* cu_k) {
  AttnArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.total_q = d.total_q;
  a.total_k = d.total_k;
  a.qs = d.q_stride;
  a.ks = d.k_stride;
  a.vs = d.v_stride;
  a.seqs = d.num_seqs;
  a.hq = d.num_heads;
  a.hk = d.num_kv_heads;
  a.group = d.num_heads / d.num_kv_heads;
  a.hd = d.head_dim;
  a.nq = static_cast<int>(d.total_q / d.num_seqs);
  a.nk = static_cast<int>(d.total_k / d.num_seqs);
  a.causal = d.causal;
  a.scale = d.scale;
  return a;
}

bool attn_vec(const msd_attn_desc& d, const AttnArgs& a, bool bwd) {
  const int64_t e = d.dtype == MSD_BF16 ? 2 : 4;
  const auto ok = [&](const void* p, int64_t stride) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * e % 16 == 0 &&
           stride <= (int64_t(1) << 22);  // a tile's rows are 32-bit offsets
  };
  return a.hd % 8 == 0 && ok(a.q, a.qs) && ok(a.k, a.ks) && ok(a.v, a.vs) &&
         (!bwd || (a.group <= 32 && int64_t(a.hq) * a.hd <= (int64_t(1) << 22)));
}

// Upper bound over both forms (packed or equal lengths): the descriptor does not say which.
size_t attn_fwd_ws_bytes(const msd_attn_desc& d) {
  const int a = splits(d, true, kNW * 32), b = splits(d, false, kNW * 32);
  const int n = a > b ? a : b, chunk = token_chunk(d);
  int64_t rows = n > 1 ? n * d.total_q : 0;
  if (chunk > 0) {
    const int64_t r = token_units(d, chunk);
    rows = rows > r ? rows : r;
  }
  return static_cast<size_t>(rows) * d.num_heads * (padded_hd(d.head_dim) + 1) * sizeof(float);
}

hipError_t launch_attn_fwd(const msd_attn_desc& d, const AttnArgs& a, void* out, void* rest,
                           float* lse, void* ws, hipStream_t s) {
  const bool vec = attn_vec(d, a, false) && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(rest) % 16 == 0;
  return d.dtype == MSD_BF16 ? launch_type<bf16>(d, a, out, rest, lse, ws, vec, s)
                             : launch_type<float>(d, a, out, nullptr, lse, ws, vec, s);
}

}  // namespace msd
