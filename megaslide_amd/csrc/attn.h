// Packed attention: arguments of the kernels and their host interface.
#pragma once

#include "common.h"

namespace msd {

struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* cu_q;  // null: equal lengths nq, nk
  const int32_t* cu_k;
  int64_t total_q, total_k;
  int64_t qs, ks, vs;   // elements between tokens
  int seqs, hq, hk, group, hd, nq, nk, causal;
  float scale;
};

struct AttnBwdPtrs {
  const void* out;
  const void* rest;  // what rounding took from out, or null
  const void* dout;
  const float* lse;
  const float* dlse;
  void* dq;
  void* dk;
  void* dv;
};

AttnArgs attn_args(const msd_attn_desc& d, const void* q, const void* k, const void* v,
                   const int32_t* cu_q, const int32_t* cu_k);
// Whether rows of q, k, v are read in 16-byte chunks (the backward: and a tile of 32 rows holds
// whole tokens of a group's heads); else element by element.
bool attn_vec(const msd_attn_desc& d, const AttnArgs& a, bool bwd);
int attn_max_head_dim();

size_t attn_fwd_ws_bytes(const msd_attn_desc& d);
hipError_t launch_attn_fwd(const msd_attn_desc& d, const AttnArgs& a, void* out, void* rest,
                           float* lse, void* ws, hipStream_t s);
size_t attn_bwd_ws_bytes(const msd_attn_desc& d);
hipError_t launch_attn_bwd(const msd_attn_desc& d, const AttnArgs& a, const AttnBwdPtrs& p,
                           void* ws, hipStream_t s);

}  // namespace msd
