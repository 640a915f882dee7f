// Elements of the three storage types (FMHC_DTYPE_*) as fp32, for the kernels
// that take more than bf16.
#pragma once

#include "fmhc_common.h"

namespace fmhc {

// load8 / store8: 8 consecutive elements at any address that is a multiple of
// the element's size, with the nontemporal hint or not; load / store: one;
// rounded: what a store leaves.  Stores round to nearest even.
template <int DT>
struct Elems;

template <>
struct Elems<FMHC_DTYPE_BF16> {
  using S = uint16_t;
  template <bool NT>
  __device__ static __forceinline__ void load8(const S* p, float f[8]) {
    unpack8(NT ? ld16_stream(p) : ld16(p), f);
  }
  template <bool NT>
  __device__ static __forceinline__ void store8(S* p, const float f[8]) {
    NT ? st16_stream(p, pack8(f)) : st16(p, pack8(f));
  }
  __device__ static __forceinline__ float load(const S* p) { return bf16_to_f32(*p); }
  __device__ static __forceinline__ void store(S* p, float v) { *p = f32_to_bf16(v); }
  __device__ static __forceinline__ float rounded(float v) { return bf16_to_f32(f32_to_bf16(v)); }
};

template <>
struct Elems<FMHC_DTYPE_F16> {
  using S = uint16_t;
  __device__ static __forceinline__ float widen(uint32_t h) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
  }
  __device__ static __forceinline__ uint16_t narrow(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
  }
  template <bool NT>
  __device__ static __forceinline__ void load8(const S* p, float f[8]) {
    const u32x4 v = NT ? ld16_stream(p) : ld16(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = widen(v[i] & 0xffffu);
      f[2 * i + 1] = widen(v[i] >> 16);
    }
  }
  template <bool NT>
  __device__ static __forceinline__ void store8(S* p, const float f[8]) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = narrow(f[2 * i]) | static_cast<uint32_t>(narrow(f[2 * i + 1])) << 16;
    NT ? st16_stream(p, v) : st16(p, v);
  }
  __device__ static __forceinline__ float load(const S* p) { return widen(*p); }
  __device__ static __forceinline__ void store(S* p, float v) { *p = narrow(v); }
  __device__ static __forceinline__ float rounded(float v) { return widen(narrow(v)); }
};

template <>
struct Elems<FMHC_DTYPE_F32> {
  using S = float;
  template <bool NT>
  __device__ static __forceinline__ void load8(const S* p, float f[8]) {
    const u32x4 a = NT ? ld16_stream(p) : ld16(p), b = NT ? ld16_stream(p + 4) : ld16(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = __uint_as_float(a[i]);
      f[4 + i] = __uint_as_float(b[i]);
    }
  }
  template <bool NT>
  __device__ static __forceinline__ void store8(S* p, const float f[8]) {
    u32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = __float_as_uint(f[i]);
      b[i] = __float_as_uint(f[4 + i]);
    }
    // Never with the hint: each of the two stores fills half of its lines.
    st16(p, a);
    st16(p + 4, b);
  }
  __device__ static __forceinline__ float load(const S* p) { return *p; }
  __device__ static __forceinline__ void store(S* p, float v) { *p = v; }
  __device__ static __forceinline__ float rounded(float v) { return v; }
};

// f(integral_constant of the type), or FMHC_ERR_INVALID_ARGUMENT.
template <typename F>
int with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case FMHC_DTYPE_F32: return f(std::integral_constant<int, FMHC_DTYPE_F32>{});
    case FMHC_DTYPE_BF16: return f(std::integral_constant<int, FMHC_DTYPE_BF16>{});
    case FMHC_DTYPE_F16: return f(std::integral_constant<int, FMHC_DTYPE_F16>{});
    default: return FMHC_ERR_INVALID_ARGUMENT;
  }
}

}  // namespace fmhc
