// Kernels of the RMS norm and of rows in 8 bits (rms_norm.hip has the entry points
// and the formulas) for one storage type; compiled once per type
// (rms_norm_{f32,bf16,f16}.hip).
#pragma once

#include "elems.h"

namespace fmhc {

struct RmsFwdArgs {
  const void* x;
  const void* r;   // added to x first; may be null
  const void* w;   // may be null (1)
  bool w_f32;      // w in fp32, otherwise in x's type
  bool norm;       // false: the rows are packed as they are (no r, no w)
  void* y;         // or null: codes
  int8_t* codes;   // rows of ld_codes bytes
  float* scales;
  int64_t ld_codes;
  void* sum;       // x + r, with r
  float* rstd;     // may be null
  int64_t T;
  int C;
  float eps;
};

struct RmsBwdArgs {
  const void* gy;
  const void* x;       // the sum where the forward had r
  const float* rstd;
  const void* w;       // may be null
  bool w_f32;          // w and gw
  const void* gi;      // a gradient of x from elsewhere, added to gx; may be null
  void* gx;
  float* partial;      // null: no gw, or few rows (rms_few)
  void* gw;            // may be null
  int64_t T;
  int C;
};

// Defined per storage type; the sizes are checked and T > 0.
template <int DT>
int rms_fwd_run(const RmsFwdArgs& a, hipStream_t s);
template <int DT>
int rms_bwd_run(const RmsBwdArgs& a, hipStream_t s);

// Workgroups of the backward, each of which leaves a sum of every column, at most.
constexpr int64_t kRmsParts = 512;
// Columns of a workgroup's sums.
inline int64_t rms_cols(int64_t C) { return (C + 7) / 8 * 8; }
// Rows that registers hold, and the partial sums at most of others, whose columns are cut into workgroups
// of 256 N: four workgroups per CU in all.
constexpr int64_t kRmsHeld = 16384;
inline int64_t rms_any_parts(int64_t T, int64_t C) {
  const int64_t each = C < 8 ? 256 : 256 * 8, blocks = (C + each - 1) / each;
  const int64_t share = 1024 / blocks > 1 ? 1024 / blocks : 1, limit = share < kRmsParts ? share : kRmsParts;
  return T < limit ? T : limit;
}

// Sums of every column that a backward leaves at most: what the workspace holds and the launches keep to.
inline int64_t rms_parts(int64_t T, int64_t C) {
  return C > kRmsHeld ? rms_any_parts(T, C) : T < kRmsParts ? T : kRmsParts;
}

// Whether grad_w of these rows is summed by workgroups of the backward's own launch, which read the rows
// again, instead of by partial sums and a second launch (one launch / two, us, bf16: T = 16 C = 1024 3.1 / 6.0,
// T = 512 3.5 / 6.4 and C = 4096 5.4 / 10.0, T = 1024 C = 1024 4.5 / 7.3, C = 2560 12.6 / 10.0, T = 2048 C = 1024
// 10.5 / 8.2).
inline bool rms_few(int64_t T, int64_t C) { return C >= 8 && C <= kRmsHeld && T <= (C <= 1024 ? 1024 : 512); }

// A row's largest magnitude counts as at least this where the row is packed.
constexpr float kRowLeast = 7.888609052210118e-31f;  // 2^-100

}  // namespace fmhc
