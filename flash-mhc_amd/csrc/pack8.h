// Block-scaled 8-bit storage of activations (pack8), shared by the kernels
// that write it and by those that read it.
//
// A row of C columns is cut into groups of 32, the last one shorter where C is
// no multiple.  A group has one scale byte E and every element one signed code:
//   a    = max |x| over the group
//   E    = clamp(exponent field of fp32(a), 7, 254);  255 where a is Inf or NaN
//   unit = 2^(E - 133)
//   code = clamp(round_half_even(x / unit), -127, 127);  0 where E = 255
// and stands for code * unit (every element of a group with E = 255 for NaN).
// With 2^e <= a < 2^(e + 1), e = E - 127, unit is 2^(e - 6): |x / unit| < 128,
// an error of at most unit / 2, a 128th of 2^e (unit at the clamp to 127).
// This is MXINT8 of the OCP microscaling formats.  x / unit is exact, so the
// codes do not depend on who computes them; code * unit has seven significant
// bits and E >= 7 keeps it out of fp32's subnormals, so it is exactly a bf16
// value: a kernel that reads codes gives what it gives on the unpacked tensor.
#pragma once

#include "fmhc_common.h"

namespace fmhc {

constexpr int kPackGroup = 32;  // columns per scale
constexpr uint32_t kPackMinE = 7, kPackMaxE = 254, kPackNan = 255;

// Scale bytes of a row of C columns.
__host__ __device__ __forceinline__ int pack_groups(int C) { return (C + kPackGroup - 1) / kPackGroup; }

// 8 codes at any byte address.
typedef unsigned int u32x2_byte __attribute__((ext_vector_type(2), aligned(1)));
template <bool NT>
__device__ __forceinline__ u32x2 ld_codes(const int8_t* p) {
#if FMHC_NT_LOADS
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x2_byte*>(p));
#endif
  return *reinterpret_cast<const u32x2_byte*>(p);
}
template <bool NT>
__device__ __forceinline__ void st_codes(int8_t* p, u32x2 v) {
#if FMHC_NT_STORES
  if constexpr (NT) return __builtin_nontemporal_store(v, reinterpret_cast<u32x2_byte*>(p));
#endif
  *reinterpret_cast<u32x2_byte*>(p) = v;
}

// unit of a scale byte: 2^(E - 133), whose exponent field is E - 6.
__device__ __forceinline__ float pack_unit(uint32_t E) {
  return __uint_as_float(E == kPackNan ? 0x7fc00000u : (E - 6u) << 23);
}

// Code I of a word as fp32.  A bit field extraction, which the compiler folds
// into the conversion's operand (from a shift and a narrowing cast it makes two
// to three instructions).
template <int I>
__device__ __forceinline__ float code_at(uint32_t w) {
  return static_cast<float>(static_cast<int>(__builtin_amdgcn_sbfe(static_cast<int>(w), 8 * I, 8)));
}

// The 8 codes as fp32.
__device__ __forceinline__ void codes8(u32x2 q, float (&f)[8]) {
  f[0] = code_at<0>(q.x), f[1] = code_at<1>(q.x), f[2] = code_at<2>(q.x), f[3] = code_at<3>(q.x);
  f[4] = code_at<0>(q.y), f[5] = code_at<1>(q.y), f[6] = code_at<2>(q.y), f[7] = code_at<3>(q.y);
}

// The values of 8 codes of one group.
__device__ __forceinline__ void decode8(u32x2 q, float unit, float (&f)[8]) {
  codes8(q, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] *= unit;
}

// The same where the group of 32 ends behind n0 columns (8 or more: all of them
// have u0).
__device__ __forceinline__ void decode8(u32x2 q, float u0, float u1, int n0, float (&f)[8]) {
  codes8(q, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] *= i < n0 ? u0 : u1;
}

// The largest magnitude's bits (NaN above Inf above every number).
__device__ __forceinline__ uint32_t max_bits8(const float f[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(f[i]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  return m;
}

// The maximum over the four lanes of a quad, which hold a group's 32 elements.
// All four must be active.
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
  // DPP controls: quad_perm [1,0,3,2], quad_perm [2,3,0,1].
  uint32_t o = __builtin_amdgcn_update_dpp(0u, m, 0xb1, 0xf, 0xf, false);
  m = o > m ? o : m;
  o = __builtin_amdgcn_update_dpp(0u, m, 0x4e, 0xf, 0xf, false);
  return o > m ? o : m;
}

__device__ __forceinline__ uint32_t pack_scale(uint32_t max_bits) {
  const uint32_t e = max_bits >> 23;
  return e == 255u ? kPackNan : e < kPackMinE ? kPackMinE : e;
}

// The codes of 8 elements of a group with scale byte E.  x / unit is a product
// with a power of two; the addition of 1.5 x 2^23 then rounds half to even and
// leaves the code in the sum's low byte.
__device__ __forceinline__ u32x2 encode8(const float f[8], uint32_t E) {
  const float inv = __uint_as_float((260u - E) << 23);
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = __builtin_amdgcn_fmed3f(f[i] * inv, -127.f, 127.f);
    b[i] = __float_as_uint(v + 12582912.f);
  }
  // Byte selectors of v_perm_b32(hi, lo): 0-3 of lo, 4-7 of hi.
  const uint32_t keep = E == kPackNan ? 0u : ~0u;
  u32x2 q;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t p = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0c0c0400u);
    const uint32_t r = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x0c0c0400u);
    q[h] = (p | r << 16) & keep;
  }
  return q;
}

// The last n codes (1 to 7) of 8, to p on: one store per bit of n.
__device__ __forceinline__ void st_last_codes(int8_t* p, u32x2 q, int n) {
  uint64_t v = (static_cast<uint64_t>(q.y) << 32 | q.x) >> (8 * (8 - n));
  typedef uint32_t u32_byte __attribute__((aligned(1)));
  typedef uint16_t u16_byte __attribute__((aligned(1)));
  if (n & 4) {
    *reinterpret_cast<u32_byte*>(p) = static_cast<uint32_t>(v);
    p += 4;
    v >>= 32;
  }
  if (n & 2) {
    *reinterpret_cast<u16_byte*>(p) = static_cast<uint16_t>(v);
    p += 2;
    v >>= 16;
  }
  if (n & 1) *p = static_cast<int8_t>(v);
}

// Where a kernel reads rows from: bf16, or codes and scales.  A Row is one row
// of C columns; load<8>(g) its element group g (8 columns), load<1>(c) one
// element.  NT: with the nontemporal hint (whole, aligned groups).  Kernels
// take `const Elem*` and the scales (unused for bf16).
struct Bf16Src {
  using Elem = uint16_t;
  static constexpr bool kPacked = false;
  template <bool NT>
  struct Row {
    const uint16_t* p;
    __device__ static __forceinline__ Row at(const Elem* x, const uint8_t*, int64_t r, int C) { return Row{x + r * C}; }
    __device__ __forceinline__ Row next(int C) const { return Row{p + C}; }
    template <int VEC>
    __device__ __forceinline__ void load(int idx, float (&f)[VEC]) const {
      Lanes<VEC, NT>::load(p, idx, f);
    }
  };
  static bool aligned(const Elem* x) { return aligned16(x); }
  // Eight columns as loaded.
  using Raw = u32x4;
  template <bool NT>
  __device__ static __forceinline__ Raw raw(const char* at) {
    return Lanes<8, NT>::raw(reinterpret_cast<const uint16_t*>(at), 0);
  }
  // Column k of token t, whose nC columns are streams of C.
  __device__ static __forceinline__ float elem(const Elem* x, const uint8_t*, int64_t t, int k, int nC, int) {
    return bf16_to_f32(x[t * nC + k]);
  }
};

struct Pack8Src {
  using Elem = int8_t;
  static constexpr bool kPacked = true;
  template <bool NT>
  struct Row {
    const int8_t* q;
    const uint8_t* s;
    __device__ static __forceinline__ Row at(const Elem* x, const uint8_t* scales, int64_t r, int C) {
      return Row{x + r * C, scales + r * pack_groups(C)};
    }
    __device__ __forceinline__ Row next(int C) const { return Row{q + C, s + pack_groups(C)}; }
    template <int VEC>
    __device__ __forceinline__ void load(int idx, float (&f)[VEC]) const {
      if constexpr (VEC == 8) {
        const u32x2 v = ld_codes<NT>(q + 8 * idx);
        decode8(v, pack_unit(s[idx >> 2]), f);
      } else {
        f[0] = static_cast<float>(q[idx]) * pack_unit(s[idx >> 5]);
      }
    }
  };
  static bool aligned(const Elem* x) { return (reinterpret_cast<uintptr_t>(x) & 7u) == 0; }
  // The scales of the eight columns' first and last element, which differ where
  // c % 8 != 0 and a group of 32 ends inside.
  struct Raw {
    u32x2 q;
    uint32_t e0, e1;
  };
  // From wave-uniform bases: the first column's code at x + off, its scale at
  // scales + soff, the last one's `step` (0 or 1) behind it.
  template <bool NT>
  __device__ static __forceinline__ Raw raw(const char* x, uint32_t off, const uint8_t* scales, uint32_t soff,
                                            uint32_t step) {
    return Raw{ld_codes<NT>(reinterpret_cast<const int8_t*>(x + off)), scales[soff], scales[soff + step]};
  }
  __device__ static __forceinline__ void widen(const Raw& v, int c, float (&f)[8]) {
    decode8(v.q, pack_unit(v.e0), pack_unit(v.e1), kPackGroup - (c & (kPackGroup - 1)), f);
  }
  __device__ static __forceinline__ float elem(const Elem* x, const uint8_t* scales, int64_t t, int k, int nC, int C) {
    const int j = k / C;
    return static_cast<float>(x[t * nC + k]) *
           pack_unit(scales[(t * (nC / C) + j) * pack_groups(C) + ((k - j * C) >> 5)]);
  }
};

// Rows of C % 8 == 0: eight columns from a multiple of 8 on have one scale.
struct Pack8WholeSrc : Pack8Src {
  struct Raw {
    u32x2 q;
    uint32_t e;
  };
  template <bool NT>
  __device__ static __forceinline__ Raw raw(const char* x, uint32_t off, const uint8_t* scales, uint32_t soff, uint32_t) {
    return Raw{ld_codes<NT>(reinterpret_cast<const int8_t*>(x + off)), scales[soff]};
  }
  __device__ static __forceinline__ void widen(const Raw& v, int, float (&f)[8]) { decode8(v.q, pack_unit(v.e), f); }
};

}  // namespace fmhc
