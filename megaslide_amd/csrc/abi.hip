// C ABI entry points: argument validation, error reporting, dispatch to the
// kernel launchers.  Declarations and conventions: include/megaslide_dsa3d.h.
#include <stdarg.h>
#include <stdio.h>

#include <mutex>

#include "attn.h"
#include "common.h"
#include "qk_rope.h"

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int launch_status(hipError_t e, const char* what) {
  if (e == hipSuccess) {
    g_err[0] = '\0';
    return MSD_OK;
  }
  return fail(MSD_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

size_t elem_bytes(int32_t dtype) { return dtype == MSD_BF16 ? 2 : 4; }

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int check_dsa(const msd_dsa3d_desc* d) {
  if (d == nullptr) return fail(MSD_ERR_ARG, "dsa3d: desc is NULL");
  if (d->B < 0 || d->T < 1 || d->H < 1 || d->W < 1)
    return fail(MSD_ERR_ARG, "dsa3d: bad shape B=%d T=%d H=%d W=%d", d->B, d->T, d->H, d->W);
  if (d->num_heads < 1 || d->head_dim < 1)
    return fail(MSD_ERR_ARG, "dsa3d: bad heads num_heads=%d head_dim=%d", d->num_heads,
                d->head_dim);
  if (d->head_dim > msd::dsa3d_max_head_dim())
    return fail(MSD_ERR_UNSUPPORTED, "dsa3d: head_dim=%d above the supported %d", d->head_dim,
                msd::dsa3d_max_head_dim());
  if (d->kt < 1 || d->kh < 1 || d->kw < 1)
    return fail(MSD_ERR_ARG, "dsa3d: bad window (%d, %d, %d)", d->kt, d->kh, d->kw);
  if (d->dtype != MSD_F32 && d->dtype != MSD_BF16)
    return fail(MSD_ERR_UNSUPPORTED, "dsa3d: dtype %d not supported", d->dtype);
  if (d->algo < MSD_ALGO_AUTO || d->algo > MSD_ALGO_TILED)
    return fail(MSD_ERR_ARG, "dsa3d: bad algo %d", d->algo);
  if (d->extra_g < 0 || d->extra_g > 4096)
    return fail(MSD_ERR_ARG, "dsa3d: extra_g %d outside [0, 4096]", d->extra_g);
  if (d->dkv_accum != MSD_ACCUM_F32 && d->dkv_accum != MSD_ACCUM_F16)
    return fail(MSD_ERR_ARG, "dsa3d: bad dkv_accum %d", d->dkv_accum);
  if (d->dkv_accum == MSD_ACCUM_F16 && d->dtype != MSD_BF16)
    return fail(MSD_ERR_ARG, "dsa3d: dkv_accum MSD_ACCUM_F16 needs bf16 storage");
  if (!(d->dropout_p >= 0.0f && d->dropout_p < 1.0f))
    return fail(MSD_ERR_ARG, "dsa3d: dropout_p %g outside [0, 1)", static_cast<double>(d->dropout_p));
  const int64_t D = static_cast<int64_t>(d->num_heads) * d->head_dim;
  if (d->q_stride < D || d->k_stride < D || d->v_stride < D)
    return fail(MSD_ERR_ARG, "dsa3d: token strides (%lld, %lld, %lld) below D=%lld",
                (long long)d->q_stride, (long long)d->k_stride, (long long)d->v_stride,
                (long long)D);
  const int64_t N = static_cast<int64_t>(d->T) * d->H * d->W;
  const int64_t C = static_cast<int64_t>(d->num_heads) * d->kt * d->kh * d->kw * 3;
  if (C > (int64_t(1) << 30) || N > (int64_t(1) << 40) || static_cast<int64_t>(d->B) * N > (int64_t(1) << 40))
    return fail(MSD_ERR_ARG, "dsa3d: sizes out of range");
  return MSD_OK;
}

int check_ptrs(const char* what, size_t align, std::initializer_list<const void*> ps) {
  int i = 0;
  for (const void* p : ps) {
    if (p == nullptr) return fail(MSD_ERR_ARG, "%s: pointer argument %d is NULL", what, i);
    if (!aligned(p, align))
      return fail(MSD_ERR_ALIGN, "%s: pointer argument %d not %zu-byte aligned", what, i, align);
    ++i;
  }
  return MSD_OK;
}

int check_conv(const msd_dwconv3d_desc* d) {
  if (d == nullptr) return fail(MSD_ERR_ARG, "dwconv3d: desc is NULL");
  if (d->B < 0 || d->T < 1 || d->H < 1 || d->W < 1 || d->C < 1)
    return fail(MSD_ERR_ARG, "dwconv3d: bad shape B=%d T=%d H=%d W=%d C=%d", d->B, d->T, d->H,
                d->W, d->C);
  if (d->kt < 1 || d->kh < 1 || d->kw < 1 || !(d->kt & 1) || !(d->kh & 1) || !(d->kw & 1))
    return fail(MSD_ERR_UNSUPPORTED, "dwconv3d: kernel (%d, %d, %d) must be odd and >= 1", d->kt,
                d->kh, d->kw);
  if (d->dtype != MSD_F32 && d->dtype != MSD_BF16)
    return fail(MSD_ERR_UNSUPPORTED, "dwconv3d: dtype %d not supported", d->dtype);
  if (d->act != 0 && d->act != 1) return fail(MSD_ERR_UNSUPPORTED, "dwconv3d: act %d", d->act);
  return MSD_OK;
}

int check_qk_rope(const msd_qk_rope_desc* d) {
  if (d == nullptr) return fail(MSD_ERR_ARG, "qk_rope: desc is NULL");
  if (d->tokens < 0 || d->tokens > (int64_t(1) << 40) || d->pos_rows < (d->tokens > 0 ? 1 : 0))
    return fail(MSD_ERR_ARG, "qk_rope: bad sizes tokens=%lld pos_rows=%lld", (long long)d->tokens,
                (long long)d->pos_rows);
  if (d->q_heads < 1 || d->k_heads < 0 || d->q_heads > 65536 || d->k_heads > 65536)
    return fail(MSD_ERR_ARG, "qk_rope: bad heads %d, %d", d->q_heads, d->k_heads);
  if (d->head_dim < 2 || d->head_dim > 256)
    return fail(MSD_ERR_UNSUPPORTED, "qk_rope: head_dim=%d outside [2, 256]", d->head_dim);
  if (d->dtype != MSD_F32 && d->dtype != MSD_BF16)
    return fail(MSD_ERR_UNSUPPORTED, "qk_rope: dtype %d not supported", d->dtype);
  if (d->norm != 0 && d->norm != 1) return fail(MSD_ERR_ARG, "qk_rope: norm %d", d->norm);
  if (d->norm && d->weight_dtype != MSD_F32 && d->weight_dtype != d->dtype)
    return fail(MSD_ERR_UNSUPPORTED, "qk_rope: weight_dtype %d with dtype %d", d->weight_dtype,
                d->dtype);
  if (d->pos_dtype < MSD_POS_I32 || d->pos_dtype > MSD_POS_GRID)
    return fail(MSD_ERR_UNSUPPORTED, "qk_rope: pos_dtype %d not supported", d->pos_dtype);
  if (d->n_axes < 1 || d->n_axes > 4)
    return fail(MSD_ERR_ARG, "qk_rope: %d axes outside [1, 4]", d->n_axes);
  if (d->pos_dtype == MSD_POS_GRID &&
      (d->n_axes != 3 ||
       (d->tokens > 0 && (d->grid[0] < 1 || d->grid[1] < 1 || d->grid[2] < 1 ||
                          d->pos_rows / d->grid[0] / d->grid[1] != d->grid[2] ||
                          d->pos_rows % d->grid[0] != 0 ||
                          d->pos_rows / d->grid[0] % d->grid[1] != 0))))
    return fail(MSD_ERR_ARG, "qk_rope: grid (%d, %d, %d) needs 3 axes and as many position rows",
                d->grid[0], d->grid[1], d->grid[2]);
  int64_t sum = 0;
  for (int x = 0; x < d->n_axes; ++x) {
    if (d->axis_dims[x] < 0 || d->axis_dims[x] % 2 != 0)
      return fail(MSD_ERR_ARG, "qk_rope: axis %d has %d channels (must be even)", x,
                  d->axis_dims[x]);
    sum += d->axis_dims[x];
  }
  if (sum > d->head_dim)
    return fail(MSD_ERR_ARG, "qk_rope: the axes' %lld channels exceed head_dim=%d", (long long)sum,
                d->head_dim);
  if (!(d->theta > 0.0) || !std::isfinite(d->theta))
    return fail(MSD_ERR_ARG, "qk_rope: theta %g must be finite and > 0", d->theta);
  if (d->norm && (!(d->eps >= 0.0f) || !std::isfinite(d->eps)))
    return fail(MSD_ERR_ARG, "qk_rope: eps %g must be finite and >= 0",
                static_cast<double>(d->eps));
  if (d->q_stride < static_cast<int64_t>(d->q_heads) * d->head_dim ||
      d->k_stride < static_cast<int64_t>(d->k_heads) * d->head_dim)
    return fail(MSD_ERR_ARG, "qk_rope: token strides (%lld, %lld) below heads*head_dim",
                (long long)d->q_stride, (long long)d->k_stride);
  return MSD_OK;
}

int check_attn(const msd_attn_desc* d) {
  if (d == nullptr) return fail(MSD_ERR_ARG, "attn: desc is NULL");
  if (d->num_heads < 1 || d->num_kv_heads < 1 || d->num_heads % d->num_kv_heads != 0)
    return fail(MSD_ERR_ARG, "attn: num_heads=%d must be a multiple of num_kv_heads=%d",
                d->num_heads, d->num_kv_heads);
  if (d->head_dim < 1 || d->head_dim > msd::attn_max_head_dim())
    return fail(MSD_ERR_UNSUPPORTED, "attn: head_dim=%d outside [1, %d]", d->head_dim,
                msd::attn_max_head_dim());
  if (d->dtype != MSD_F32 && d->dtype != MSD_BF16)
    return fail(MSD_ERR_UNSUPPORTED, "attn: dtype %d not supported", d->dtype);
  if (d->causal != 0 && d->causal != 1) return fail(MSD_ERR_ARG, "attn: causal %d", d->causal);
  if (d->num_seqs < 1) return fail(MSD_ERR_ARG, "attn: num_seqs=%d", d->num_seqs);
  // rows are counted in 32 bits; a launch has below 2^24 workgroups of 256 threads: one for each
  // 128 rows and one a sequence and head
  constexpr int64_t kMost = int64_t(1) << 30;
  if (d->total_q < 0 || d->total_k < 0 || d->num_heads > 65536 ||
      d->num_seqs > (kMost >> 8) / d->num_heads ||
      d->total_q > kMost / d->num_heads || d->total_k > kMost / d->num_kv_heads)
    return fail(MSD_ERR_ARG, "attn: sizes out of range (total_q=%lld, total_k=%lld, num_seqs=%d)",
                (long long)d->total_q, (long long)d->total_k, d->num_seqs);
  if (!(d->scale > 0.0f) || !std::isfinite(d->scale))
    return fail(MSD_ERR_ARG, "attn: scale %g must be finite and > 0",
                static_cast<double>(d->scale));
  const int64_t dq = static_cast<int64_t>(d->num_heads) * d->head_dim;
  const int64_t dk = static_cast<int64_t>(d->num_kv_heads) * d->head_dim;
  if (d->q_stride < dq || d->k_stride < dk || d->v_stride < dk)
    return fail(MSD_ERR_ARG, "attn: strides (%lld, %lld, %lld) below heads*head_dim",
                (long long)d->q_stride, (long long)d->k_stride, (long long)d->v_stride);
  return MSD_OK;
}

int check_lengths(const msd_attn_desc* d, const int32_t* cu_q, const int32_t* cu_k) {
  if ((cu_q == nullptr) != (cu_k == nullptr))
    return fail(MSD_ERR_ARG, "attn: cu_q and cu_k go together");
  if (cu_q != nullptr && (!aligned(cu_q, 4) || !aligned(cu_k, 4)))
    return fail(MSD_ERR_ALIGN, "attn: cu_q or cu_k not 4-byte aligned");
  if (cu_q == nullptr && (d->total_q % d->num_seqs != 0 || d->total_k % d->num_seqs != 0))
    return fail(MSD_ERR_ARG, "attn: totals %lld, %lld are no multiples of num_seqs=%d",
                (long long)d->total_q, (long long)d->total_k, d->num_seqs);
  return MSD_OK;
}

// Scratch of msd_dsa3d_bwd_noalloc: one array on every GPU that loads the
// library, held until the process ends.  Host code never passes the array's
// name (a host-side stand-in) to a kernel: it uses the per-device address that
// hipGetSymbolAddress returns.  Calls that overlap on one GPU share it and race.
constexpr size_t kNoAllocScratchBytes = MSD_NOALLOC_SCRATCH_BYTES;
static __device__ __align__(256) unsigned char scratch[kNoAllocScratchBytes];

constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;
void* g_scratch[kMaxDevices] = {};

// Device address of `scratch` on the current device, looked up once per device
// with that device current.
int scratch_address(void** out) {
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess)
    return fail(MSD_ERR_LAUNCH, "dsa3d_bwd_noalloc: hipGetDevice: %s", hipGetErrorString(e));
  if (dev < 0 || dev >= kMaxDevices)
    return fail(MSD_ERR_UNSUPPORTED, "dsa3d_bwd_noalloc: device %d beyond the %d supported", dev,
                kMaxDevices);
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (g_scratch[dev] == nullptr) {
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess || p == nullptr)
      return fail(MSD_ERR_LAUNCH, "dsa3d_bwd_noalloc: hipGetSymbolAddress(scratch): %s",
                  hipGetErrorString(e));
    g_scratch[dev] = p;
  }
  *out = g_scratch[dev];
  return MSD_OK;
}

int dsa3d_bwd_impl(const msd_dsa3d_desc* desc, const void* q, const void* k, const void* v,
                   const void* offsets, const void* ek, const void* ev, const void* out,
                   const void* dout, const float* lse, const float* dlse, void* dq, void* dk,
                   void* dv, void* doffsets, void* dek, void* dev, void* workspace,
                   size_t workspace_bytes, void* stream, bool noalloc) {
  int rc = check_dsa(desc);
  if (rc != MSD_OK) return rc;
  rc = check_ptrs("dsa3d_bwd", elem_bytes(desc->dtype),
                  {q, k, v, offsets, out, dout, dq, dk, dv, doffsets});
  if (rc != MSD_OK) return rc;
  if (desc->extra_g > 0) {
    rc = check_ptrs("dsa3d_bwd(extra_k, extra_v, d_extra_k, d_extra_v)", 16, {ek, ev, dek, dev});
    if (rc != MSD_OK) return rc;
  }
  rc = check_ptrs("dsa3d_bwd(lse)", 4, {lse});
  if (rc != MSD_OK) return rc;
  if (dlse != nullptr && !aligned(dlse, 4)) return fail(MSD_ERR_ALIGN, "dsa3d_bwd: dlse misaligned");
  if (desc->B == 0) return MSD_OK;
  const size_t need = msd::dsa3d_bwd_ws_bytes(*desc);
  if (noalloc) {
    if (need > kNoAllocScratchBytes)
      return fail(MSD_ERR_WORKSPACE,
                  "dsa3d_bwd_noalloc: the call needs %zu bytes of scratch, above the %zu-byte "
                  "maximum of the no-allocation entry point (use msd_dsa3d_bwd with a workspace)",
                  need, kNoAllocScratchBytes);
    rc = scratch_address(&workspace);
    if (rc != MSD_OK) return rc;
    workspace_bytes = kNoAllocScratchBytes;
  }
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(MSD_ERR_WORKSPACE, "dsa3d_bwd: workspace of %zu bytes (16-aligned) needed, got %zu",
                need, workspace == nullptr ? size_t(0) : workspace_bytes);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  // the tiled backward also writes dq with 16-byte rows and reads out/dout rows of D
  const bool tiled_ok = msd::dsa3d_tiled_supported(*desc, q, k, v) &&
                        msd::dsa3d_tiled_supported(*desc, dq, dk, dv);
  if (desc->algo == MSD_ALGO_TILED && !tiled_ok)
    return fail(MSD_ERR_UNSUPPORTED,
                "dsa3d_bwd: tiled kernels need bf16 or fp32, head_dim 32, 64, 96 or 128, <= 160 taps, "
                "<= 256 extra keys, 16-byte aligned rows and samples that 32-bit row offsets address");
  if (tiled_ok && desc->algo != MSD_ALGO_DIRECT)
    return launch_status(msd::launch_dsa3d_bwd_tiled(*desc, q, k, v, offsets, ek, ev, out, dout,
                                                     lse, dlse, dq, dk, dv, doffsets, dek, dev,
                                                     workspace, s),
                         "dsa3d_bwd");
  // head sizes between the compiled ones: on padded copies, where the workspace
  // holds them
  if (msd::dsa3d_ragged_supported(*desc, q, k, v) &&
      workspace_bytes >= msd::dsa3d_ragged_bwd_ws_bytes(*desc))
    return launch_status(msd::launch_dsa3d_bwd_ragged(*desc, q, k, v, offsets, ek, ev, out, dout,
                                                      lse, dlse, dq, dk, dv, doffsets, dek, dev,
                                                      workspace, s),
                         "dsa3d_bwd");
  return launch_status(msd::launch_dsa3d_bwd_direct(*desc, q, k, v, offsets, ek, ev, out, dout,
                                                    lse, dlse, dq, dk, dv, doffsets, dek, dev,
                                                    workspace, s),
                       "dsa3d_bwd");
}

}  // namespace

extern "C" {

int msd_abi_version(void) { return MSD_ABI_VERSION; }

const char* msd_last_error(void) { return g_err; }

int msd_dsa3d_fwd(const msd_dsa3d_desc* desc, const void* q, const void* k, const void* v,
                  const void* offsets, const void* extra_k, const void* extra_v, void* out,
                  float* lse, void* stream) {
  int rc = check_dsa(desc);
  if (rc != MSD_OK) return rc;
  rc = check_ptrs("dsa3d_fwd", elem_bytes(desc->dtype), {q, k, v, offsets, out});
  if (rc != MSD_OK) return rc;
  if (desc->extra_g > 0) {
    rc = check_ptrs("dsa3d_fwd(extra_k, extra_v)", 16, {extra_k, extra_v});
    if (rc != MSD_OK) return rc;
  }
  if (lse != nullptr && !aligned(lse, 4)) return fail(MSD_ERR_ALIGN, "dsa3d_fwd: lse misaligned");
  const bool tiled_ok = msd::dsa3d_tiled_supported(*desc, q, k, v);
  if (desc->algo == MSD_ALGO_TILED && !tiled_ok)
    return fail(MSD_ERR_UNSUPPORTED,
                "dsa3d_fwd: tiled kernels need bf16 or fp32, head_dim 32, 64, 96 or 128, <= 160 taps, "
                "<= 256 extra keys, 16-byte aligned rows and samples that 32-bit row offsets address");
  if (desc->B == 0) return MSD_OK;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (tiled_ok && desc->algo != MSD_ALGO_DIRECT)
    return launch_status(msd::launch_dsa3d_fwd_tiled(*desc, q, k, v, offsets, extra_k, extra_v,
                                                     out, lse, s),
                         "dsa3d_fwd");
  if (msd::dsa3d_ragged_supported(*desc, q, k, v))
    return launch_status(msd::launch_dsa3d_fwd_ragged(*desc, q, k, v, offsets, extra_k, extra_v,
                                                      out, lse, s),
                         "dsa3d_fwd");
  return launch_status(msd::launch_dsa3d_fwd_direct(*desc, q, k, v, offsets, extra_k, extra_v, out,
                                                    lse, s),
                       "dsa3d_fwd");
}

size_t msd_dsa3d_bwd_workspace_size(const msd_dsa3d_desc* desc) {
  if (check_dsa(desc) != MSD_OK) return 0;
  return msd::dsa3d_bwd_ws_bytes(*desc);
}

size_t msd_dsa3d_bwd_best_workspace_size(const msd_dsa3d_desc* desc) {
  if (check_dsa(desc) != MSD_OK) return 0;
  const size_t need = msd::dsa3d_bwd_ws_bytes(*desc);
  if (!msd::dsa3d_ragged_supported(*desc, nullptr, nullptr, nullptr)) return need;
  const size_t ragged = msd::dsa3d_ragged_bwd_ws_bytes(*desc);
  return ragged > need ? ragged : need;
}

int msd_dsa3d_bwd(const msd_dsa3d_desc* desc, const void* q, const void* k, const void* v,
                  const void* offsets, const void* extra_k, const void* extra_v, const void* out,
                  const void* dout, const float* lse, const float* dlse, void* dq, void* dk,
                  void* dv, void* doffsets, void* d_extra_k, void* d_extra_v, void* workspace,
                  size_t workspace_bytes, void* stream) {
  return dsa3d_bwd_impl(desc, q, k, v, offsets, extra_k, extra_v, out, dout, lse, dlse, dq, dk, dv,
                        doffsets, d_extra_k, d_extra_v, workspace, workspace_bytes, stream, false);
}

int msd_dsa3d_bwd_noalloc(const msd_dsa3d_desc* desc, const void* q, const void* k,
                          const void* v, const void* offsets, const void* extra_k,
                          const void* extra_v, const void* out, const void* dout,
                          const float* lse, const float* dlse, void* dq, void* dk, void* dv,
                          void* doffsets, void* d_extra_k, void* d_extra_v, void* stream) {
  return dsa3d_bwd_impl(desc, q, k, v, offsets, extra_k, extra_v, out, dout, lse, dlse, dq, dk, dv,
                        doffsets, d_extra_k, d_extra_v, nullptr, 0, stream, true);
}

int msd_dwconv3d_fwd(const msd_dwconv3d_desc* desc, const void* x, const void* weight,
                     const void* bias, void* y, void* preact, void* stream) {
  int rc = check_conv(desc);
  if (rc != MSD_OK) return rc;
  const size_t a = elem_bytes(desc->dtype);
  rc = check_ptrs("dwconv3d_fwd", a, {x, weight, y});
  if (rc != MSD_OK) return rc;
  for (const void* p : {static_cast<const void*>(bias), static_cast<const void*>(preact)})
    if (p != nullptr && !aligned(p, a)) return fail(MSD_ERR_ALIGN, "dwconv3d_fwd: misaligned");
  if (preact != nullptr && desc->act != 1)
    return fail(MSD_ERR_ARG, "dwconv3d_fwd: preact is the GELU input (act = 1 only)");
  if (desc->B == 0) return MSD_OK;
  return launch_status(msd::launch_dwconv3d_fwd(*desc, x, weight, bias, y, preact,
                                                static_cast<hipStream_t>(stream)),
                       "dwconv3d_fwd");
}

size_t msd_dwconv3d_bwd_workspace_size(const msd_dwconv3d_desc* desc) {
  if (check_conv(desc) != MSD_OK) return 0;
  return msd::dwconv3d_bwd_ws_bytes(*desc);
}

int msd_dwconv3d_bwd(const msd_dwconv3d_desc* desc, const void* x, const void* weight,
                     const void* bias, const void* preact, const void* dy, void* dx,
                     void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                     void* stream) {
  int rc = check_conv(desc);
  if (rc != MSD_OK) return rc;
  const size_t a = elem_bytes(desc->dtype);
  rc = check_ptrs("dwconv3d_bwd", a, {x, weight, dy});
  if (rc != MSD_OK) return rc;
  for (const void* p : {static_cast<const void*>(bias), static_cast<const void*>(dx),
                        static_cast<const void*>(dweight), static_cast<const void*>(dbias),
                        preact})
    if (p != nullptr && !aligned(p, a)) return fail(MSD_ERR_ALIGN, "dwconv3d_bwd: misaligned");
  if (preact != nullptr && desc->act != 1)
    return fail(MSD_ERR_ARG, "dwconv3d_bwd: preact is the GELU input (act = 1 only)");
  if (desc->B == 0) return MSD_OK;
  const size_t need = msd::dwconv3d_bwd_ws_bytes(*desc);
  if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16))
    return fail(MSD_ERR_WORKSPACE,
                "dwconv3d_bwd: workspace of %zu bytes (16-aligned) needed, got %zu", need,
                workspace == nullptr ? size_t(0) : workspace_bytes);
  return launch_status(msd::launch_dwconv3d_bwd(*desc, x, weight, bias, preact, dy, dx, dweight,
                                                dbias, workspace, static_cast<hipStream_t>(stream)),
                       "dwconv3d_bwd");
}

int msd_qk_rope_fwd(const msd_qk_rope_desc* desc, const void* q, const void* k,
                    const void* q_weight, const void* k_weight, const void* positions,
                    void* q_out, void* k_out, void* stream) {
  int rc = check_qk_rope(desc);
  if (rc != MSD_OK) return rc;
  if (desc->tokens == 0) return MSD_OK;
  const size_t a = elem_bytes(desc->dtype);
  rc = check_ptrs("qk_rope_fwd", a, {q, q_out});
  if (rc == MSD_OK && desc->k_heads > 0) rc = check_ptrs("qk_rope_fwd(k)", a, {k, k_out});
  if (rc == MSD_OK && desc->pos_dtype != MSD_POS_GRID)
    rc = check_ptrs("qk_rope_fwd(positions)", desc->pos_dtype & 1 ? 8 : 4, {positions});
  if (rc != MSD_OK) return rc;
  for (const void* p : {q_weight, k_weight})
    if (p != nullptr && !aligned(p, elem_bytes(desc->weight_dtype)))
      return fail(MSD_ERR_ALIGN, "qk_rope_fwd: weight misaligned");
  const msd::QkRopePtrs p{{q, k}, {q_weight, k_weight}, {}, {q_out, k_out}, {}, positions};
  return launch_status(
      msd::launch_qk_rope(*desc, p, false, nullptr, static_cast<hipStream_t>(stream)),
      "qk_rope_fwd");
}

size_t msd_qk_rope_bwd_workspace_size(const msd_qk_rope_desc* desc) {
  if (check_qk_rope(desc) != MSD_OK) return 0;
  return msd::qk_rope_bwd_ws_bytes(*desc);
}

int msd_qk_rope_bwd(const msd_qk_rope_desc* desc, const void* q, const void* k,
                    const void* q_weight, const void* k_weight, const void* positions,
                    const void* dq_out, const void* dk_out, void* dq, void* dk, void* dq_weight,
                    void* dk_weight, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_qk_rope(desc);
  if (rc != MSD_OK) return rc;
  const size_t a = elem_bytes(desc->dtype);
  if (desc->tokens > 0) {
    rc = check_ptrs("qk_rope_bwd", a, {dq_out, dq});
    if (rc == MSD_OK && desc->k_heads > 0) rc = check_ptrs("qk_rope_bwd(k)", a, {dk_out, dk});
    if (rc == MSD_OK && desc->norm) rc = check_ptrs("qk_rope_bwd(q)", a, {q});
    if (rc == MSD_OK && desc->norm && desc->k_heads > 0)
      rc = check_ptrs("qk_rope_bwd(k input)", a, {k});
    if (rc == MSD_OK && desc->pos_dtype != MSD_POS_GRID)
      rc = check_ptrs("qk_rope_bwd(positions)", desc->pos_dtype & 1 ? 8 : 4, {positions});
    if (rc != MSD_OK) return rc;
  }
  for (const void* p : {q_weight, k_weight, static_cast<const void*>(dq_weight),
                        static_cast<const void*>(dk_weight)})
    if (p != nullptr && !aligned(p, elem_bytes(desc->weight_dtype)))
      return fail(MSD_ERR_ALIGN, "qk_rope_bwd: weight misaligned");
  if (dk_weight != nullptr && desc->k_heads == 0)
    return fail(MSD_ERR_ARG, "qk_rope_bwd: dk_weight without k");
  const size_t need = msd::qk_rope_bwd_ws_bytes(*desc);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(MSD_ERR_WORKSPACE,
                "qk_rope_bwd: workspace of %zu bytes (16-aligned) needed, got %zu", need,
                workspace == nullptr ? size_t(0) : workspace_bytes);
  const msd::QkRopePtrs p{{q, k}, {q_weight, k_weight}, {dq_out, dk_out}, {dq, dk},
                          {dq_weight, dk_weight}, positions};
  return launch_status(
      msd::launch_qk_rope(*desc, p, true, workspace, static_cast<hipStream_t>(stream)),
      "qk_rope_bwd");
}

size_t msd_attn_fwd_workspace_size(const msd_attn_desc* desc) {
  if (check_attn(desc) != MSD_OK) return 0;
  return msd::attn_fwd_ws_bytes(*desc);
}

int msd_attn_fwd(const msd_attn_desc* desc, const void* q, const void* k, const void* v,
                 const int32_t* cu_q, const int32_t* cu_k, void* out, void* out_rest, float* lse,
                 void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_attn(desc);
  if (rc == MSD_OK) rc = check_lengths(desc, cu_q, cu_k);
  if (rc != MSD_OK) return rc;
  if (desc->total_q == 0) return MSD_OK;
  const size_t a = elem_bytes(desc->dtype);
  rc = check_ptrs("attn_fwd", a, {q, out});
  if (rc == MSD_OK && desc->total_k > 0) rc = check_ptrs("attn_fwd(k, v)", a, {k, v});
  if (rc != MSD_OK) return rc;
  if (lse != nullptr && !aligned(lse, 4)) return fail(MSD_ERR_ALIGN, "attn_fwd: lse misaligned");
  if (out_rest != nullptr && (!aligned(out_rest, a) || desc->dtype != MSD_BF16))
    return fail(MSD_ERR_ARG, "attn_fwd: out_rest misaligned or not of bf16 results");
  const size_t need = msd::attn_fwd_ws_bytes(*desc);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(MSD_ERR_WORKSPACE, "attn_fwd: workspace of %zu bytes (16-aligned) needed, got %zu",
                need, workspace == nullptr ? size_t(0) : workspace_bytes);
  return launch_status(msd::launch_attn_fwd(*desc, msd::attn_args(*desc, q, k, v, cu_q, cu_k), out,
                                            out_rest, lse, workspace,
                                            static_cast<hipStream_t>(stream)),
                       "attn_fwd");
}

size_t msd_attn_bwd_workspace_size(const msd_attn_desc* desc) {
  if (check_attn(desc) != MSD_OK) return 0;
  return msd::attn_bwd_ws_bytes(*desc);
}

int msd_attn_bwd(const msd_attn_desc* desc, const void* q, const void* k, const void* v,
                 const int32_t* cu_q, const int32_t* cu_k, const void* out, const void* out_rest,
                 const void* dout, const float* lse, const float* dlse, void* dq, void* dk,
                 void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_attn(desc);
  if (rc == MSD_OK) rc = check_lengths(desc, cu_q, cu_k);
  if (rc != MSD_OK) return rc;
  const size_t a = elem_bytes(desc->dtype);
  if (desc->total_q > 0) {
    rc = check_ptrs("attn_bwd", a, {q, out, dout, dq});
    if (rc == MSD_OK) rc = check_ptrs("attn_bwd(lse)", 4, {lse});
  }
  if (rc == MSD_OK && desc->total_k > 0) rc = check_ptrs("attn_bwd(k, v)", a, {k, v, dk, dv});
  if (rc != MSD_OK) return rc;
  if (dlse != nullptr && !aligned(dlse, 4)) return fail(MSD_ERR_ALIGN, "attn_bwd: dlse misaligned");
  if (out_rest != nullptr && (!aligned(out_rest, a) || desc->dtype != MSD_BF16))
    return fail(MSD_ERR_ARG, "attn_bwd: out_rest misaligned or not of bf16 results");
  const size_t need = msd::attn_bwd_ws_bytes(*desc);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(MSD_ERR_WORKSPACE, "attn_bwd: workspace of %zu bytes (16-aligned) needed, got %zu",
                need, workspace == nullptr ? size_t(0) : workspace_bytes);
  const msd::AttnBwdPtrs p{out, out_rest, dout, lse, dlse, dq, dk, dv};
  return launch_status(msd::launch_attn_bwd(*desc, msd::attn_args(*desc, q, k, v, cu_q, cu_k), p,
                                            workspace, static_cast<hipStream_t>(stream)),
                       "attn_bwd");
}

}  // extern "C"
