// pack8 and unpack8: a tensor's rows to block-scaled 8 bits and back (pack8.h
// has the format).
//
// A lane holds 8 consecutive columns, a quad of lanes a group of 32, so the
// group's maximum takes two cross-lane moves and no LDS; one pass over the
// data, no atomics.  Bound by HBM: a bf16 element is 2 bytes one way and
// 33/32 the other, some 6 VALU operations.
#include "elems.h"
#include "pack8.h"

namespace fmhc {

namespace {

// Lane i of a launch: row i / (4 G), group (i / 4) % G, quarter i % 4 of it.
// FLAT: C % 32 == 0, the tensor taken as one row (no division).  A launch
// covers at most 2^31 lanes.
struct Place {
  int64_t elem;   // first element of the lane's 8
  int64_t group;  // its scale byte
  int n;          // columns of the 8 inside the row (at most 8; 0 or less: none)
};
template <bool FLAT>
__device__ __forceinline__ Place place_of(uint32_t i, int C, uint32_t G) {
  const uint32_t grp = i >> 2, q = i & 3u;
  if constexpr (FLAT) {
    return Place{int64_t{i} * 8, grp, 8};
  } else {
    const uint32_t r = grp / G, g = grp - r * G;
    const int c = static_cast<int>(32u * g + 8u * q);
    return Place{int64_t{r} * C + c, grp, C - c};
  }
}

template <int DT, bool FLAT>
__global__ __launch_bounds__(256) void pack8_kernel(const typename Elems<DT>::S* __restrict__ x,
                                                    int8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                    uint32_t lanes, int C, uint32_t G) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= lanes) return;  // whole quads
  const Place p = place_of<FLAT>(i, C, G);
  float f[8];
  if (FLAT || p.n >= 8) {
    Elems<DT>::template load8<true>(x + p.elem, f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < p.n ? Elems<DT>::load(x + p.elem + e) : 0.f;
  }
  const uint32_t E = pack_scale(quad_max(max_bits8(f)));
  const u32x2 q = encode8(f, E);
  if (FLAT || p.n >= 8) {
    st_codes<FLAT>(codes + p.elem, q);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < p.n) codes[p.elem + e] = static_cast<int8_t>(q[e >> 2] >> (8 * (e & 3)));
  }
  if ((i & 3u) == 0) scales[p.group] = static_cast<uint8_t>(E);
}

template <int DT, bool FLAT>
__global__ __launch_bounds__(256) void unpack8_kernel(const int8_t* __restrict__ codes,
                                                      const uint8_t* __restrict__ scales,
                                                      typename Elems<DT>::S* __restrict__ x, uint32_t lanes, int C,
                                                      uint32_t G) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= lanes) return;
  const Place p = place_of<FLAT>(i, C, G);
  const float unit = pack_unit(scales[p.group]);
  if (FLAT || p.n >= 8) {
    float f[8];
    decode8(ld_codes<FLAT>(codes + p.elem), unit, f);
    Elems<DT>::template store8<true>(x + p.elem, f);
  } else {
    for (int e = 0; e < p.n; ++e) Elems<DT>::store(x + p.elem + e, static_cast<float>(codes[p.elem + e]) * unit);
  }
}

bool bad_sizes(int64_t rows, int64_t C) {
  return rows < 0 || C <= 0 || C > (int64_t{1} << 30) || rows > (int64_t{1} << 62) / (C + 32);
}

// f(first row, rows, lanes) over pieces of at most 2^31 lanes.
template <typename F>
void for_pieces(int64_t rows, int64_t C, F&& f) {
  const int64_t per_row = 4 * ((C + kPackGroup - 1) / kPackGroup);
  const int64_t most = (int64_t{1} << 31) / per_row;  // C <= 2^30: at least 16
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    f(r, static_cast<uint32_t>(n * per_row));
  }
}

}  // namespace
}  // namespace fmhc

extern "C" int fmhc_pack8(const void* x, int dtype, int8_t* codes, uint8_t* scales, int64_t rows, int64_t C,
                          void* stream) {
  using namespace fmhc;
  if (bad_sizes(rows, C)) return FMHC_ERR_INVALID_ARGUMENT;
  return with_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (rows == 0) return FMHC_OK;
    if (!x || !codes || !scales) return FMHC_ERR_INVALID_ARGUMENT;
    const auto* xs = static_cast<const typename Elems<DT>::S*>(x);
    const int c = static_cast<int>(C), G = pack_groups(c);
    for_pieces(rows, C, [&](int64_t r, uint32_t lanes) {
      auto launch = [&](auto flat) {
        pack8_kernel<DT, decltype(flat)::value><<<dim3(blocks_for(lanes, 256)), 256, 0, static_cast<hipStream_t>(stream)>>>(
            xs + r * C, codes + r * C, scales + r * G, lanes, c, static_cast<uint32_t>(G));
      };
      C % kPackGroup == 0 ? launch(std::true_type{}) : launch(std::false_type{});
    });
    return launch_status();
  });
}

extern "C" int fmhc_unpack8(const int8_t* codes, const uint8_t* scales, void* x, int dtype, int64_t rows, int64_t C,
                            void* stream) {
  using namespace fmhc;
  if (bad_sizes(rows, C)) return FMHC_ERR_INVALID_ARGUMENT;
  return with_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (rows == 0) return FMHC_OK;
    if (!x || !codes || !scales) return FMHC_ERR_INVALID_ARGUMENT;
    auto* xs = static_cast<typename Elems<DT>::S*>(x);
    const int c = static_cast<int>(C), G = pack_groups(c);
    for_pieces(rows, C, [&](int64_t r, uint32_t lanes) {
      auto launch = [&](auto flat) {
        unpack8_kernel<DT, decltype(flat)::value><<<dim3(blocks_for(lanes, 256)), 256, 0, static_cast<hipStream_t>(stream)>>>(
            codes + r * C, scales + r * G, xs + r * C, lanes, c, static_cast<uint32_t>(G));
      };
      C % kPackGroup == 0 ? launch(std::true_type{}) : launch(std::false_type{});
    });
    return launch_status();
  });
}
