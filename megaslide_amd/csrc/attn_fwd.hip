// Attention over packed sequences, forward: out = softmax(scale q k^T + mask) v.
//
// Rows of a workgroup are (query token, head of the group) pairs of one key head, so a tile of
// keys and values is read once for all heads that share it; one token's heads are rows of one
// block.  One pass over the keys with the running maximum m and sum l of a softmax (fp32):
// S^T = K Q^T, p = exp2(c (s - m)), O^T += V^T P^T, each a block of the matrix cores with the
// rows along the lanes, so that m, l and the rescale of O are one value a lane and P is a
// fragment where it stands.  m is raised only where a score exceeds it by 2^8 or more in p
// (p <= 256: nothing is lost in fp32), which spares most rescales.
#include "attn_common.h"

namespace msd {
namespace {

constexpr int kBN = 64;  // keys of a tile

template <typename T, int HD, int NW, bool VEC>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 ? (HD <= 64 ? 4 : 2) : 1) void attn_fwd_kernel(
    const AttnArgs a, T* __restrict__ out, float* __restrict__ lse, float* __restrict__ part,
    int nsplit) {
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
  std::conditional_t<kDma, TileDma<HD, kBN, kNT>, Tile<T, HD, kBN, kNT, VEC>> tk, tv;
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
    if (lse != nullptr && g == 0) lse[at_row] = ls;
  }
}

// Joins the parts of rows whose keys were split: out = sum_i exp(lse_i - lse) out_i.  One wave
// a row.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(const float* __restrict__ part,
                                                        int nsplit, int64_t rows, int hd,
                                                        int stride, T* __restrict__ out,
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
    if (lane + 64 * x < hd) out[row * hd + lane + 64 * x] = from_f32<T>(acc[x] * inv);
  if (lse != nullptr && lane == 0) lse[row] = sum == 0.0f ? -INFINITY : base + logf(sum);
}

int padded_hd(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 96 ? 96 : 128; }

int64_t q_slots(const msd_attn_desc& d, bool packed, int tile) {
  const int64_t group = d.num_heads / d.num_kv_heads;
  if (!packed) return d.total_q / d.num_seqs == 0 ? 0 : d.num_seqs * ((d.total_q / d.num_seqs * group + tile - 1) / tile);
  return d.total_q * group / tile + d.num_seqs + 1;
}

// Workgroups along the keys: enough that the launch fills the 256 compute units several times,
// each with 256 keys at least of a sequence of mean length.
int splits(const msd_attn_desc& d, bool packed, int tile) {
  const int64_t wgs = q_slots(d, packed, tile) * d.num_kv_heads;
  if (wgs == 0 || wgs >= 512) return 1;
  const int64_t mean = d.total_k / d.num_seqs;
  int64_t n = (1024 + wgs - 1) / wgs;
  const int64_t most = (mean + 255) / 256;
  n = n < most ? n : most;
  return static_cast<int>(n < 1 ? 1 : n > 256 ? 256 : n);
}

constexpr int kNW = 4;

template <typename T, int HD>
hipError_t launch_hd(const msd_attn_desc& d, const AttnArgs& a, T* out, float* lse, float* ws,
                     bool vec, hipStream_t s) {
  const bool packed = a.cu_q != nullptr;
  const int n = splits(d, packed, kNW * 32);
  const int64_t slots = q_slots(d, packed, kNW * 32);
  const int64_t blocks = slots * n * a.hk;
  if (blocks == 0) return hipSuccess;
  if (vec)
    attn_fwd_kernel<T, HD, kNW, true>
        <<<static_cast<unsigned>(blocks), kNW * 64, 0, s>>>(a, out, lse, ws, n);
  else
    attn_fwd_kernel<T, HD, kNW, false>
        <<<static_cast<unsigned>(blocks), kNW * 64, 0, s>>>(a, out, lse, ws, n);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || n == 1) return e;
  const int64_t rows = a.total_q * a.hq;
  attn_join_kernel<T><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, s>>>(ws, n, rows, a.hd, HD,
                                                                           out, lse);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const msd_attn_desc& d, const AttnArgs& a, void* out, float* lse, void* ws,
                       bool vec, hipStream_t s) {
  T* o = static_cast<T*>(out);
  float* w = static_cast<float*>(ws);
  switch (padded_hd(a.hd)) {
    case 32: return launch_hd<T, 32>(d, a, o, lse, w, vec, s);
    case 64: return launch_hd<T, 64>(d, a, o, lse, w, vec, s);
    case 96: return launch_hd<T, 96>(d, a, o, lse, w, vec, s);
    default: return launch_hd<T, 128>(d, a, o, lse, w, vec, s);
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
           stride <= (int64_t(1) << 23);  // a tile's rows are 32-bit offsets
  };
  return a.hd % 8 == 0 && ok(a.q, a.qs) && ok(a.k, a.ks) && ok(a.v, a.vs) &&
         (!bwd || (a.group <= 32 && int64_t(a.hq) * a.hd <= (int64_t(1) << 23)));
}

// Upper bound over both forms (packed or equal lengths): the descriptor does not say which.
size_t attn_fwd_ws_bytes(const msd_attn_desc& d) {
  const int a = splits(d, true, kNW * 32), b = splits(d, false, kNW * 32);
  const int n = a > b ? a : b;
  if (n == 1) return 0;
  return static_cast<size_t>(n) * d.total_q * d.num_heads * (padded_hd(d.head_dim) + 1) *
         sizeof(float);
}

hipError_t launch_attn_fwd(const msd_attn_desc& d, const AttnArgs& a, void* out, float* lse,
                           void* ws, hipStream_t s) {
  const bool vec = attn_vec(d, a, false) && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  return d.dtype == MSD_BF16 ? launch_type<bf16>(d, a, out, lse, ws, vec, s)
                             : launch_type<float>(d, a, out, lse, ws, vec, s);
}

}  // namespace msd
