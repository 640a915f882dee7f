// Layer norm over the last axis, forward and backward, with the input kept as
// it is or in 8 bits (pack8.h) for the backward: the C entry points.
//
//   forward   mean = sum_c x / C,  rstd = rsqrt(sum_c (x - mean)^2 / C + eps)
//             y = h w + b,  h = (x - mean) rstd
//   backward  g = gy w,  h = (x' - mean) rstd   (x' is x, or what its codes stand for)
//             grad_x = rstd (g - sum_c g / C - h sum_c g h / C)   (+ x's gradient from elsewhere)
//             grad_w = sum_t gy h,  grad_b = sum_t gy
//
// Everything is fp32 but the stored tensors, each rounded once.  The variance is
// taken around the mean (no difference of large sums) with the row in
// registers, so x is read once.  The workgroups' sums of grad_w and grad_b are
// added by a second kernel in a fixed order (no atomics: deterministic).  The
// kernels are in layer_norm_kernels.h.
#include "layer_norm.h"

namespace fmhc {

namespace {

// Zero gradients of the parameters of an empty batch (a kernel, not a memset,
// so that the call can be captured in a graph).
__global__ __launch_bounds__(256) void ln_zero_kernel(uint16_t* __restrict__ p, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}

int64_t ln_workspace(int64_t T, int64_t C) {
  return (T < kLnParts ? T : kLnParts) * 2 * ln_cols(C) * static_cast<int64_t>(sizeof(float));
}

bool bad_sizes(int64_t T, int64_t C) {
  return T < 0 || C <= 0 || C > (int64_t{1} << 28) || T > (int64_t{1} << 60) / C;
}

// The parameters are fp32 or of x's type.
bool bad_types(int dtype, int param_dtype) {
  if (dtype != FMHC_DTYPE_F32 && dtype != FMHC_DTYPE_BF16 && dtype != FMHC_DTYPE_F16) return true;
  return param_dtype != FMHC_DTYPE_F32 && param_dtype != dtype;
}

}  // namespace

extern template int ln_fwd_run<FMHC_DTYPE_F32>(const LnFwdArgs&, hipStream_t);
extern template int ln_fwd_run<FMHC_DTYPE_BF16>(const LnFwdArgs&, hipStream_t);
extern template int ln_fwd_run<FMHC_DTYPE_F16>(const LnFwdArgs&, hipStream_t);
extern template int ln_bwd_run<FMHC_DTYPE_F32>(const LnBwdArgs&, hipStream_t);
extern template int ln_bwd_run<FMHC_DTYPE_BF16>(const LnBwdArgs&, hipStream_t);
extern template int ln_bwd_run<FMHC_DTYPE_F16>(const LnBwdArgs&, hipStream_t);

}  // namespace fmhc

extern "C" int fmhc_layer_norm_fwd(const void* x, const void* weight, const void* bias, void* y, float* mean,
                                   float* rstd, int8_t* x_codes, uint8_t* x_scales, int dtype, int param_dtype,
                                   int64_t T, int64_t C, float eps, void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C) || bad_types(dtype, param_dtype) || !x_codes != !x_scales) return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (!x || !y) return FMHC_ERR_INVALID_ARGUMENT;
  const LnFwdArgs a{x,       LnParams{weight, bias, param_dtype == FMHC_DTYPE_F32}, y, mean, rstd, x_codes, x_scales, T,
                    static_cast<int>(C), eps};
  return with_dtype(dtype, [&](auto dt) { return ln_fwd_run<decltype(dt)::value>(a, static_cast<hipStream_t>(stream)); });
}

extern "C" int64_t fmhc_layer_norm_bwd_workspace_bytes(int64_t T, int64_t C) {
  if (fmhc::bad_sizes(T, C) || T == 0) return 0;
  return fmhc::ln_workspace(T, C);
}

extern "C" int fmhc_layer_norm_bwd(const void* grad_y, const void* x, const int8_t* x_codes, const uint8_t* x_scales,
                                   const float* mean, const float* rstd, const void* weight,
                                   const void* grad_x_in, void* grad_x, void* grad_weight, void* grad_bias,
                                   void* workspace, int64_t workspace_bytes, int dtype, int param_dtype, int64_t T,
                                   int64_t C, void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C) || bad_types(dtype, param_dtype) || !x_codes != !x_scales || (x && x_codes) ||
      (grad_x_in && grad_x_in == grad_x))
    return FMHC_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f32 = param_dtype == FMHC_DTYPE_F32;
  if (T == 0) {
    const int64_t n = C * (f32 ? 2 : 1);  // 16-bit words of a parameter's gradient
    for (void* p : {grad_weight, grad_bias})
      if (p) ln_zero_kernel<<<dim3(blocks_for(n, 256)), 256, 0, s>>>(static_cast<uint16_t*>(p), n);
    return launch_status();
  }
  if (!grad_y || (!x && !x_codes) || !mean || !rstd || !grad_x) return FMHC_ERR_INVALID_ARGUMENT;
  const bool params = grad_weight || grad_bias;
  if (params && (!workspace || workspace_bytes < ln_workspace(T, C) || !aligned16(workspace)))
    return FMHC_ERR_INVALID_ARGUMENT;
  const LnBwdArgs a{grad_y, x,      x_codes, x_scales, mean, rstd, LnParams{weight, nullptr, f32}, grad_x_in, grad_x,
                    params ? static_cast<float*>(workspace) : nullptr, grad_weight, grad_bias, T, static_cast<int>(C)};
  return with_dtype(dtype, [&](auto dt) { return ln_bwd_run<decltype(dt)::value>(a, s); });
}
