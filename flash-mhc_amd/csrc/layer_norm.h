// Kernels of the layer norm (layer_norm.hip has the entry points and the
// formulas) and how rows are laid over lanes, for one storage type; compiled
// once per type (layer_norm_{f32,bf16,f16}.hip).
#pragma once

#include <type_traits>

#include "elems.h"
#include "pack8.h"

namespace fmhc {

// The norm's weight and bias, in fp32 or x's type; either may be null (1, 0).
struct LnParams {
  const void* w;
  const void* b;
  bool f32;
};

struct LnFwdArgs {
  const void* x;
  LnParams P;
  void* y;
  float* mean;      // may be null
  float* rstd;      // may be null
  int8_t* codes;    // null: x is not packed
  uint8_t* scales;
  int64_t T;
  int C;
  float eps;
};

struct LnBwdArgs {
  const void* gy;
  const void* x;         // null: from codes and scales
  const int8_t* codes;
  const uint8_t* scales;
  const float* mean;
  const float* rstd;
  LnParams P;            // b unused
  const void* gi;        // a gradient of x from elsewhere, added to gx; may be null
  void* gx;
  float* partial;        // null: no parameter gradients
  void* gw;              // may be null
  void* gb;              // may be null
  int64_t T;
  int C;
};

// Defined per storage type; the sizes are checked and T > 0.
template <int DT>
int ln_fwd_run(const LnFwdArgs& a, hipStream_t s);
template <int DT>
int ln_bwd_run(const LnBwdArgs& a, hipStream_t s);

// Workgroups of the backward, each of which leaves sums of all columns, at most:
// one of eight waves per CU, two where a lane has one group of columns and the
// registers for them (T = 65536, C = 512 one 41.4 us, two 39.8; C = 2048, two groups
// per lane, one 135, two 140, with twice as many sums to add).
constexpr int64_t kLnParts = 512;
// Columns of a workgroup's sums.
inline int64_t ln_cols(int64_t C) { return (C + 7) / 8 * 8; }

}  // namespace fmhc
