// Host interface of qk_rope.hip.
#pragma once

#include "common.h"

namespace msd {

struct QkRopePtrs {
  const void* x[2];   // q, k
  const void* w[2];   // norm weights (may be null)
  const void* dy[2];  // backward: gradients of the results
  void* y[2];         // forward: results; backward: gradients of q, k
  void* dw[2];        // backward: gradients of the weights (may be null)
  const void* pos;
};

size_t qk_rope_bwd_ws_bytes(const msd_qk_rope_desc& d);
hipError_t launch_qk_rope(const msd_qk_rope_desc& d, const QkRopePtrs& p, bool bwd, void* ws,
                          hipStream_t s);

}  // namespace msd
