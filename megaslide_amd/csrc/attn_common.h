// Device helpers of the packed attention kernels (attn_fwd.hip, attn_bwd.hip): which rows a
// workgroup has, tiles in LDS, matrix-core fragments.
//
// All products are 32x32 blocks of the matrix cores.  A fragment is 8 consecutive values of the
// summed index for one row (A) or column (B) a lane: lane l has row l % 32 and half g = l / 32
// of 16 summed values (bf16: one instruction; fp32: eight, the same layout, since the order of
// summed indexes is free as long as A and B agree).  A result block has column l % 32 in lane
// l, rows 8 (r / 4) + 4 g + r % 4 in its 16 registers.  So a block of weights computed with its
// queries (or keys) along the lanes is itself, rounded, a fragment of the next product over its
// register rows: {4 g + 0..3, 8 + 4 g + 0..3} of each 16, and no lane exchanges anything.  The
// other operand of that product is read from the row-major tile by transposing LDS reads.
#pragma once

#include "attn.h"
#include "common.h"

#include <type_traits>

namespace msd {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634074f;
constexpr float kLn2 = 0.69314718055994530942f;

// ---------------------------------------------------------------------------
// element types
// ---------------------------------------------------------------------------

template <typename T>
struct Elem;

template <>
struct Elem<bf16> {
  typedef bf16x8 frag;
  static constexpr int kPerChunk = 8;  // elements of 16 bytes
};
template <>
struct Elem<float> {
  typedef f32x8 frag;
  static constexpr int kPerChunk = 4;
};

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// Registers 8 t .. 8 t + 7 of a block of weights as a fragment (bf16: rounded to nearest even,
// half a step of 2^-8 relative, the one rounding between the two products).
template <typename T>
__device__ __forceinline__ typename Elem<T>::frag to_frag(const f32x16& s, int t) {
  typename Elem<T>::frag r;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (sizeof(T) == 2)
      r[j] = static_cast<__bf16>(s[8 * t + j]);
    else
      r[j] = s[8 * t + j];
  }
  return r;
}

template <typename F>
__device__ __forceinline__ F zero_frag() {
  F r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = 0;
  return r;
}

// Which places are masked is decided by comparing indexes, never by adding a large number, so a
// masked score may be NaN.  In the products over rows (P V and those of the gradients) a masked
// place has weight zero, but zero times an infinity or NaN is NaN: tiles that a causal mask cuts
// enter those products by their finite part, and what was left out is noted in `seen_bad`
// (nonzero) and added afterwards where it is seen.
struct FiniteBf16 {
  uint32_t found = 0;

  __device__ __forceinline__ bf16x8 operator()(const bf16x8& f) {
    u32x4 u = __builtin_bit_cast(u32x4, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // a half's bit 15 where its exponent is all ones, then the half's mask
      const uint32_t b = ((u[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
      found |= b;
      u[i] &= ~(b | (b - (b >> 15)));
    }
    return __builtin_bit_cast(bf16x8, u);
  }
  __device__ __forceinline__ bool bad() const { return found != 0; }
};
struct FiniteF32 {
  bool any = false;

  __device__ __forceinline__ f32x8 operator()(const f32x8& f) {
    f32x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool fin = fabsf(f[j]) < INFINITY;
      any |= !fin;
      r[j] = fin ? f[j] : 0.0f;
    }
    return r;
  }
  __device__ __forceinline__ bool bad() const { return any; }
};
template <typename T>
using Finite = std::conditional_t<sizeof(T) == 2, FiniteBf16, FiniteF32>;

// Maximum and sum of a value over the two halves of a wave (lanes l and l ^ 32).
__device__ __forceinline__ float half_max(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);  // lower, upper half's
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---------------------------------------------------------------------------
// sequences
// ---------------------------------------------------------------------------

struct Span {
  int64_t q0, k0;  // first row of the sequence's queries and keys
  int lq, lk;
  int seq;         // the number of sequences: rows behind the last one
  int tile;        // tile of this workgroup within the sequence; < 0: no work
};

__device__ __forceinline__ int64_t bound_of(const int32_t* cu, int s, int64_t total) {
  if (s == 0) return 0;
  const int64_t c = cu[s];
  return c < 0 ? 0 : (c > total ? total : c);
}

// Sum (or maximum) of a wave's values, in every lane's reach: lane 63 has it after the DPP steps
// within rows of 16 lanes and the two broadcasts across them.
template <bool MAX>
__device__ __forceinline__ int wave_reduce(int x) {
  const auto step = [&](int y) { x = MAX ? (x > y ? x : y) : x + y; };
  step(__builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8
  step(__builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // row_bcast 15, 31
  step(__builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}

// The sequence and tile of work item `slot`, where a sequence of n rows (times `mul`) takes
// tiles of `tile` rows.  There are floor(mul total / tile) + sequences + 1 slots: at least as
// many as tiles, and a number that is known on the host from the totals alone, so lengths stay
// on the device.  Rows behind the last sequence make one more sequence without a counterpart.
// Offsets that are not in order or out of range give wrong rows, never rows outside the tensors.
// `keys`: tiles of keys, else of queries.
//
// Workgroups start in the order of their slots, so the tiles with the most work come first and
// the last ones to end are short: with up to 63 sequences (one a lane) by what a causal mask
// leaves of them, or by their sequence's length, each wave finds its tile with a few reductions.
// More sequences keep their own order, sequence s from slot floor(mul cu[s] / tile) + s on.
__device__ __forceinline__ Span find_span(const AttnArgs& a, int slot, int mul, int tile,
                                          bool keys) {
  Span r;
  const int32_t* cu = keys ? a.cu_k : a.cu_q;
  const int64_t total = keys ? a.total_k : a.total_q;
  const int lane = threadIdx.x & 63;
  int s;
  if (cu == nullptr) {
    const int n = keys ? a.nk : a.nq;
    const int per = static_cast<int>((static_cast<int64_t>(n) * mul + tile - 1) / tile);
    s = slot % a.seqs;
    r.tile = keys ? slot / a.seqs : per - 1 - slot / a.seqs;
  } else if (a.seqs < 64) {
    const int64_t c0 = lane < a.seqs ? bound_of(cu, lane, total) : 0;
    const int64_t c1 = lane < a.seqs ? bound_of(cu, lane + 1, total) : 0;
    const int len = static_cast<int>(c1 > c0 ? c1 - c0 : 0);
    const int nt = static_cast<int>((static_cast<int64_t>(len) * mul + tile - 1) / tile);
    const int all = wave_reduce<false>(nt);
    if (slot >= all) {
      s = a.seqs;
      r.tile = slot - all;
    } else if (a.causal) {
      // tiles by levels, from the highest: level v has tile v of the queries (the last - v of
      // the keys) of every sequence that has so many
      const int most = wave_reduce<true>(nt);
      int lo = 0, hi = most - 1, above = 0;  // the lowest level with at most `slot` tiles above
      while (lo < hi) {
        const int v = (lo + hi) / 2;
        if (wave_reduce<false>(nt > v + 1 ? nt - v - 1 : 0) <= slot)
          hi = v;
        else
          lo = v + 1;
      }
      above = wave_reduce<false>(nt > lo + 1 ? nt - lo - 1 : 0);
      uint64_t with = __ballot(nt > lo);
      for (int k = slot - above; k > 0; --k) with &= with - 1;
      s = __builtin_ctzll(with | (uint64_t(1) << 63));
      r.tile = keys ? __builtin_amdgcn_readlane(nt, s) - 1 - lo : lo;
    } else {
      int before = 0;  // tiles of longer sequences, and of earlier ones of the same length
      for (int i = 0; i < a.seqs; ++i) {
        const int l = __builtin_amdgcn_readlane(len, i);
        if (l > len || (l == len && i < lane)) before += __builtin_amdgcn_readlane(nt, i);
      }
      const uint64_t here = __ballot(lane < a.seqs && slot >= before && slot < before + nt);
      s = __builtin_ctzll(here | (uint64_t(1) << 63));
      r.tile = slot - __builtin_amdgcn_readlane(before, s);
    }
    s = s < a.seqs ? s : a.seqs;
  } else {
    int lo = 0, n = a.seqs + 1;  // the answer is in [lo, lo + n)
    int64_t first = 0;           // its first slot
    while (n > 1) {
      const int step = (n + 63) / 64;
      const int i = lane * step;
      const bool in = i < n;
      const int64_t c = in ? bound_of(cu, lo + i, total) * mul / tile + lo + i : 0;
      const uint64_t ok = __ballot(in && c <= slot);
      const int k = ok == 0 ? 0 : 63 - __builtin_clzll(ok);
      first = __shfl(c, k);
      lo += k * step;
      n = n - k * step < step ? n - k * step : step;
    }
    s = __builtin_amdgcn_readfirstlane(lo);
    r.tile = __builtin_amdgcn_readfirstlane(static_cast<int>(slot - first));
  }
  const bool tail = s >= a.seqs;
  r.seq = s;
  if (a.cu_q != nullptr) {
    r.q0 = tail && keys ? 0 : bound_of(a.cu_q, s, a.total_q);
    int64_t e = tail ? (keys ? 0 : a.total_q) : bound_of(a.cu_q, s + 1, a.total_q);
    r.lq = static_cast<int>(e > r.q0 ? e - r.q0 : 0);
  } else {
    r.q0 = static_cast<int64_t>(s) * a.nq;
    r.lq = tail ? 0 : a.nq;
  }
  if (a.cu_k != nullptr) {
    r.k0 = tail && !keys ? 0 : bound_of(a.cu_k, s, a.total_k);
    int64_t e = tail ? (keys ? a.total_k : 0) : bound_of(a.cu_k, s + 1, a.total_k);
    r.lk = static_cast<int>(e > r.k0 ? e - r.k0 : 0);
  } else {
    r.k0 = static_cast<int64_t>(s) * a.nk;
    r.lk = tail ? 0 : a.nk;
  }
  r.q0 = (static_cast<int64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(r.q0))));
  r.k0 = (static_cast<int64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(r.k0))));
  r.lq = __builtin_amdgcn_readfirstlane(r.lq);
  r.lk = __builtin_amdgcn_readfirstlane(r.lk);
  const int64_t rows = static_cast<int64_t>(keys ? r.lk : r.lq) * mul;
  if (r.tile < 0 || static_cast<int64_t>(r.tile) * tile >= rows) r.tile = -1;
  return r;
}

// The tiles [first, end) of number `split` of `nsplit` workgroups that share `tiles` tiles.
__device__ __forceinline__ void split_range(int tiles, int nsplit, int split, int* first,
                                            int* end) {
  const int per = (tiles + nsplit - 1) / nsplit;
  *first = split * per < tiles ? split * per : tiles;
  *end = *first + per < tiles ? *first + per : tiles;
}

// ---------------------------------------------------------------------------
// tiles
// ---------------------------------------------------------------------------

// XOR of a row's 16-byte chunks.  bf16: sixteen rows at one chunk (16-byte reads) and four rows
// at four chunks (transposing reads) fill the 64 banks once.  fp32: eight rows at one chunk do.
template <typename T, int HD>
__device__ __forceinline__ int swz(int row) {
  if (sizeof(T) == 4) return row & 7;
  const int k = (row >> 2) & 3;
  if (HD == 128) return ((row & 3) << 2) | k;
  if (HD == 64) return (((row >> 1) & 1) << 2) | k;
  return k;
}

// Element offset of channel c (a multiple of a chunk's) of a tile's row.
template <typename T, int HD>
__device__ __forceinline__ int at(int row, int c) {
  constexpr int E = Elem<T>::kPerChunk;
  return row * HD + (((c / E) ^ swz<T, HD>(row)) * E) + c % E;
}

// A tile of ROWS rows of HD channels on its way from memory to LDS, NT threads.  Rows at or
// past `rows` and channels at or past hd become zeros.  VEC: 16-byte loads (aligned rows, hd a
// multiple of a chunk).
template <typename T, int HD, int ROWS, int NT, bool VEC>
struct Tile {
  static constexpr int E = Elem<T>::kPerChunk;
  static constexpr int kChunks = HD / E;
  static constexpr int kItems = (ROWS * kChunks + NT - 1) / NT;
  u32x4 r[kItems];

  template <typename RowPtr>
  __device__ __forceinline__ void load(RowPtr row_ptr, int rows, int hd) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int item = threadIdx.x + i * NT;
      const int row = item / kChunks, c = item % kChunks * E;
      u32x4 v = {0, 0, 0, 0};
      if (row < rows && row < ROWS && c < hd) {
        const T* p = row_ptr(row, i) + c;
        if (VEC) {
          v = *reinterpret_cast<const u32x4*>(p);
        } else if (sizeof(T) == 2) {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (c + j < hd) v[j / 2] |= static_cast<uint32_t>(h[j]) << (16 * (j & 1));
        } else {
          const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + j < hd) v[j] = w[j];
        }
      }
      r[i] = v;
    }
  }

  __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int item = threadIdx.x + i * NT;
      const int row = item / kChunks, c = item % kChunks * E;
      if (ROWS * kChunks % NT == 0 || row < ROWS)
        *reinterpret_cast<u32x4*>(lds + at<T, HD>(row, c)) = r[i];
    }
  }
};

// The same tile straight from memory to LDS, 16 bytes a lane, without registers on the way.  A
// wave's lanes fill 1,024 bytes of LDS in lane order; the XOR of the chunks is in which chunk a lane
// reads.  A row at or past `rows` (of one stride each, or the last one of row_off's) and channels
// at or past hd lie behind the buffer's end and arrive as zeros.  NT: threads that share a tile, a
// workgroup's or (64) one wave's.
template <typename T, int HD, int ROWS, int NT>
struct TileDma {
  static constexpr int E = Elem<T>::kPerChunk;
  static constexpr int kChunks = HD / E;
  static constexpr int kItems = (ROWS * kChunks + NT - 1) / NT;
  static_assert(ROWS * kChunks % 64 == 0, "whole waves");
  uint32_t voff[kItems];

  // row_off(r): element offset of row r from the tile's first, below 2^29; negative: no row
  template <typename RowOff>
  __device__ __forceinline__ void init(int hd, RowOff row_off) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int item = static_cast<int>(threadIdx.x) % NT + i * NT;
      const int row = item / kChunks;
      const int c = (item % kChunks ^ swz<T, HD>(row)) * E;
      const int64_t off = row_off(row);
      voff[i] = off < 0 || c >= hd ? 0x80000000u : static_cast<uint32_t>(off + c) * sizeof(T);
    }
  }

  // p: the tile's first row, the same in every lane; bytes: from p to the end of its last row
  __device__ __forceinline__ void issue(const T* p, int64_t bytes, const T* lds) const {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    const uint32_t n = bytes < 0 ? 0u : bytes > 0x7fffffff ? 0x7fffffffu : static_cast<uint32_t>(bytes);
    u32x4 rsrc = {static_cast<uint32_t>(at), static_cast<uint32_t>(at >> 32) & 0xffffu, n,
                  0x00020000u};
#pragma unroll
    for (int i = 0; i < 4; ++i) rsrc[i] = __builtin_amdgcn_readfirstlane(rsrc[i]);
    const uint32_t base = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) T*)lds)));
    const uint32_t wave =
        NT == 64 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (ROWS * kChunks % NT != 0 && wave + i * NT * 16 >= ROWS * HD * sizeof(T)) break;
      // writes LDS only: no register is an output (nothing else here uses m0); waited for by
      // dma_wait
      asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :
                   : "s"(base + wave + i * NT * 16), "v"(voff[i]), "s"(rsrc)
                   : "memory");
    }
  }
};

// Waits for this wave's loads to LDS but the N latest; a barrier afterwards makes them everyone's.
template <int N = 0>
__device__ __forceinline__ void dma_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// 8 channels c .. c + 7 (c a multiple of 8) of a tile's row.
template <typename T, int HD>
__device__ __forceinline__ typename Elem<T>::frag row_frag(const T* lds, int row, int c) {
  if constexpr (sizeof(T) == 2) {
    return *reinterpret_cast<const bf16x8*>(lds + at<T, HD>(row, c));
  } else {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(lds + at<T, HD>(row, c));
    const f32x4 hi = *reinterpret_cast<const f32x4*>(lds + at<T, HD>(row, c + 4));
    return f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
}

// Channel 32 blk + l % 32 of the tile's rows r0 + {4 g + 0..3, 8 + 4 g + 0..3} (r0 a multiple
// of 16): the fragment that goes with to_frag's.
template <typename T, int HD>
__device__ __forceinline__ typename Elem<T>::frag col_frag(T* lds, int r0, int blk) {
  const int l = threadIdx.x & 63, g = l >> 5;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((address_space(3))) bf16x4 lds4;
    const int row = r0 + 4 * g + ((l & 15) >> 2);
    const int c = blk * 32 + ((l >> 4) & 1) * 16 + (l & 3) * 4;
    const T* p = lds + at<T, HD>(row, c & ~7) + (c & 7);
    const T* q = lds + at<T, HD>(row + 8, c & ~7) + (c & 7);
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4*)p);
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4*)q);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const int c = blk * 32 + (l & 31);
    f32x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int row = r0 + (j / 4) * 8 + 4 * g + j % 4;
      r[j] = lds[at<T, HD>(row, c & ~3) + (c & 3)];
    }
    return r;
  }
}

// 8 channels of a row in memory, zeros at or past hd.
template <typename T, bool VEC>
__device__ __forceinline__ typename Elem<T>::frag mem_frag(const T* p, int c, int hd) {
  typename Elem<T>::frag r = zero_frag<typename Elem<T>::frag>();
  if (VEC) {
    if (c < hd) {
      if constexpr (sizeof(T) == 2) {
        r = *reinterpret_cast<const bf16x8*>(p + c);
      } else {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(p + c);
        const f32x4 hi = *reinterpret_cast<const f32x4*>(p + c + 4);
        r = f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (c + j < hd) {
        if constexpr (sizeof(T) == 2)
          r[j] = reinterpret_cast<const __bf16*>(p)[c + j];
        else
          r[j] = p[c + j];
      }
    }
  }
  return r;
}

// Stores block `blk` (32 channels) of a result with rows along the lanes: out[c] of the lane's
// row, times f.
template <typename T, bool VEC>
__device__ __forceinline__ void store_block(T* out, const f32x16& acc, int blk, float f, int hd) {
  const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = blk * 32 + 8 * i + 4 * g;
    if (VEC) {
      if (c < hd) {
        if constexpr (sizeof(T) == 2) {
          bf16x4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = static_cast<__bf16>(acc[4 * i + j] * f);
          *reinterpret_cast<bf16x4*>(out + c) = v;
        } else {
          *reinterpret_cast<f32x4*>(out + c) = f32x4{acc[4 * i] * f, acc[4 * i + 1] * f,
                                                     acc[4 * i + 2] * f, acc[4 * i + 3] * f};
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < hd) out[c + j] = from_f32<T>(acc[4 * i + j] * f);
    }
  }
}

// What rounding to bf16 took from a result, rounded itself: the backward's delta = sum(dO O)
// multiplies every weight of its row, and from the rounded result alone it would be off by as
// much as the weights' own rounding.
template <typename T>
__device__ __forceinline__ float rest_of(float v) {
  return sizeof(T) == 2 ? v - static_cast<float>(static_cast<__bf16>(v)) : 0.0f;
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_rest(T* out, const f32x16& acc, int blk, float f, int hd) {
  f32x16 r;
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = rest_of<T>(acc[i] * f);
  store_block<T, VEC>(out, r, blk, 1.0f, hd);
}

// Adds the infinities and NaN of rows [r0, r1) (r0 <= r1; row_ptr(r): row r) to a result with
// channels in its registers, for the rows that seen(r) of this lane: what was left out of a
// product by Finite.  A weight at a place that is not masked is positive, or NaN and then the
// result is NaN already, so a sum over the seen infinities and NaN is the product's.  Rare: plain
// loads, one row at a time.
template <typename T, int BLK, typename RowPtr, typename Seen>
__device__ __forceinline__ void add_nonfinite(f32x16 (&acc)[BLK], int r0, int r1, int hd,
                                           RowPtr row_ptr, Seen seen) {
  const int g = (threadIdx.x >> 5) & 1;
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    const T* p = row_ptr(r);
    if (!seen(r)) continue;
#pragma unroll
    for (int b = 0; b < BLK; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = b * 32 + 8 * (i / 4) + 4 * g + i % 4;
        const float x = c < hd ? to_f32(p[c]) : 0.0f;
        if (!(fabsf(x) < INFINITY)) acc[b][i] += x;
      }
  }
}

}  // namespace msd
