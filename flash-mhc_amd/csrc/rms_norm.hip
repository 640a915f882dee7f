// RMS norm over the last axis, forward and backward, with the residual's addition,
// and rows in 8 bits: the C entry points.
//
//   forward   s = round(x + r)   (x where there is no r)
//             rstd = rsqrt(sum_c s^2 / C + eps),  y = s rstd w
//   packed    top = max(max_c |y|, 2^-100),  scale = top / 127,  code = round_half_even(y / scale)
//   backward  g = gy w,  h = s rstd
//             grad_x = rstd (g - h sum_c g h / C)   (+ s's gradient from elsewhere)
//             grad_w = sum_t gy h
//
// Everything is fp32 but the stored tensors, each rounded once; r's gradient is
// x's.  grad_w of many rows is added from the workgroups' sums by a second kernel,
// that of few rows by workgroups of their own; in a fixed order (no atomics:
// deterministic).  The kernels are in rms_norm_kernels.h.
#include "rms_norm.h"

namespace fmhc {

namespace {

// The zero gradient of an empty batch (a kernel, not a memset, so that the call can
// be captured in a graph).
__global__ __launch_bounds__(256) void rms_zero_kernel(uint16_t* __restrict__ p, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}

int64_t rms_workspace(int64_t T, int64_t C) {
  if (rms_few(T, C)) return 0;
  return rms_parts(T, C) * rms_cols(C) * static_cast<int64_t>(sizeof(float));
}

bool bad_sizes(int64_t T, int64_t C) {
  return T < 0 || C <= 0 || C > (int64_t{1} << 28) || T > (int64_t{1} << 60) / C;
}

bool bad_type(int dtype) { return dtype != FMHC_DTYPE_F32 && dtype != FMHC_DTYPE_BF16 && dtype != FMHC_DTYPE_F16; }

// The weight is fp32 or of x's type.
bool bad_types(int dtype, int param_dtype) {
  return bad_type(dtype) || (param_dtype != FMHC_DTYPE_F32 && param_dtype != dtype);
}

bool bad_pitch(int64_t T, int64_t C, int64_t ld) { return ld < C || ld > (int64_t{1} << 60) / (T > 0 ? T : 1); }

int forward(const RmsFwdArgs& a, int dtype, void* stream) {
  return with_dtype(dtype, [&](auto dt) { return rms_fwd_run<decltype(dt)::value>(a, static_cast<hipStream_t>(stream)); });
}

}  // namespace

extern template int rms_fwd_run<FMHC_DTYPE_F32>(const RmsFwdArgs&, hipStream_t);
extern template int rms_fwd_run<FMHC_DTYPE_BF16>(const RmsFwdArgs&, hipStream_t);
extern template int rms_fwd_run<FMHC_DTYPE_F16>(const RmsFwdArgs&, hipStream_t);
extern template int rms_bwd_run<FMHC_DTYPE_F32>(const RmsBwdArgs&, hipStream_t);
extern template int rms_bwd_run<FMHC_DTYPE_BF16>(const RmsBwdArgs&, hipStream_t);
extern template int rms_bwd_run<FMHC_DTYPE_F16>(const RmsBwdArgs&, hipStream_t);

}  // namespace fmhc

extern "C" int fmhc_rms_norm_fwd(const void* x, const void* residual, const void* weight, void* y, void* sum,
                                 float* rstd, int dtype, int param_dtype, int64_t T, int64_t C, float eps,
                                 void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C) || bad_types(dtype, param_dtype) || !residual != !sum) return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (!x || !y) return FMHC_ERR_INVALID_ARGUMENT;
  return forward(RmsFwdArgs{x, residual, weight, param_dtype == FMHC_DTYPE_F32, true, y, nullptr, nullptr, 0, sum, rstd,
                            T, static_cast<int>(C), eps},
                 dtype, stream);
}

extern "C" int fmhc_rms_norm_pack8_rows(const void* x, const void* residual, const void* weight, int8_t* codes,
                                        float* scales, void* sum, int dtype, int param_dtype, int64_t T, int64_t C,
                                        int64_t ld_codes, float eps, void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C) || bad_types(dtype, param_dtype) || bad_pitch(T, C, ld_codes) || !residual != !sum)
    return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (!x || !codes || !scales) return FMHC_ERR_INVALID_ARGUMENT;
  return forward(RmsFwdArgs{x, residual, weight, param_dtype == FMHC_DTYPE_F32, true, nullptr, codes, scales, ld_codes,
                            sum, nullptr, T, static_cast<int>(C), eps},
                 dtype, stream);
}

extern "C" int fmhc_pack8_rows(const void* x, int dtype, int8_t* codes, float* scales, int64_t rows, int64_t C,
                               int64_t ld_codes, void* stream) {
  using namespace fmhc;
  if (bad_sizes(rows, C) || bad_type(dtype) || bad_pitch(rows, C, ld_codes)) return FMHC_ERR_INVALID_ARGUMENT;
  if (rows == 0) return FMHC_OK;
  if (!x || !codes || !scales) return FMHC_ERR_INVALID_ARGUMENT;
  return forward(RmsFwdArgs{x, nullptr, nullptr, true, false, nullptr, codes, scales, ld_codes, nullptr, nullptr, rows,
                            static_cast<int>(C), 0.f},
                 dtype, stream);
}

extern "C" int64_t fmhc_rms_norm_bwd_workspace_bytes(int64_t T, int64_t C) {
  if (fmhc::bad_sizes(T, C) || T == 0) return 0;
  return fmhc::rms_workspace(T, C);
}

extern "C" int fmhc_rms_norm_bwd(const void* grad_y, const void* x, const float* rstd, const void* weight,
                                 const void* grad_x_in, void* grad_x, void* grad_weight, void* workspace,
                                 int64_t workspace_bytes, int dtype, int param_dtype, int64_t T, int64_t C,
                                 void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C) || bad_types(dtype, param_dtype)) return FMHC_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f32 = param_dtype == FMHC_DTYPE_F32;
  if (T == 0) {
    const int64_t n = C * (f32 ? 2 : 1);  // 16-bit words of the weight's gradient
    if (grad_weight) rms_zero_kernel<<<dim3(blocks_for(n, 256)), 256, 0, s>>>(static_cast<uint16_t*>(grad_weight), n);
    return launch_status();
  }
  if (!grad_y || !x || !rstd || !grad_x || (grad_x_in && grad_x_in == grad_x)) return FMHC_ERR_INVALID_ARGUMENT;
  const int64_t need = grad_weight ? rms_workspace(T, C) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return FMHC_ERR_INVALID_ARGUMENT;
  // (grad_w's workgroups read grad_y and x while others store grad_x, or after it.)
  if (grad_x == grad_y || grad_x == x) return FMHC_ERR_INVALID_ARGUMENT;
  const RmsBwdArgs a{grad_y, x, rstd, weight, f32, grad_x_in, grad_x,
                     need > 0 ? static_cast<float*>(workspace) : nullptr, grad_weight, T, static_cast<int>(C)};
  return with_dtype(dtype, [&](auto dt) { return rms_bwd_run<decltype(dt)::value>(a, s); });
}
