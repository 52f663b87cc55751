// What the recurrent forms of the KDA layer share (kda_decode.cu, kda_tree.cu): short quotients and the checks of a call's
// arguments.
#pragma once

#include "common.cuh"
#include "ops.h"

namespace ssb {

SSB_DEVICE float sigmoid_fast(float z) { return __fdividef(1.0f, 1.0f + exp_fast(-z)); }
SSB_DEVICE float silu_fast(float y) { return __fdividef(y, 1.0f + exp_fast(-y)); }
SSB_DEVICE float2 bf2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }

inline bool kda_aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
// What the launches have in common: the state, the layer's parameters and the inputs.
inline bool kda_step_args(const KdaArgs& a) {
  // empty tensors (no rows, no sequences) have no address
  if ((a.T > 0 && (a.x == nullptr || a.g == nullptr || a.beta == nullptr)) || (a.R > 0 && a.seqs == nullptr) ||
      a.a_log == nullptr || a.dt_bias == nullptr || a.conv_w == nullptr || a.conv_state == nullptr ||
      a.rec_state == nullptr || a.T < 0 || a.T > 0x7fffffff || (a.cs_stride % 2) || (a.rs_stride % 4) ||
      a.cs_stride < 9 * (int64_t)a.P || a.rs_stride < (int64_t)a.H * 128 * 128 || !kda_aligned(a.x, 4) ||
      !kda_aligned(a.g, 4) || !kda_aligned(a.conv_w, 16) || !kda_aligned(a.dt_bias, 8) || !kda_aligned(a.conv_state, 4) ||
      !kda_aligned(a.rec_state, 16) || !kda_aligned(a.seqs, 16) || !kda_aligned(a.beta, 2))
    return false;
  // one row has no pitch: what the caller's tensors state there is not used
  return a.T <= 1 || (a.ldx % 2 == 0 && a.ldg % 2 == 0 && a.ldx >= 3 * (int64_t)a.P && a.ldg >= a.P && a.ldb >= a.H);
}

}  // namespace ssb
