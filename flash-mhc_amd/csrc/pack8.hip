// pack8 and unpack8: a tensor's rows to block-scaled 8 bits and back (pack8.h
// has the format).
//
// A lane holds 8 consecutive columns, a quad of lanes a group of 32, so the
// group's maximum takes two cross-lane moves and no LDS; one pass over the
// data, no atomics.  Bound by HBM: a bf16 element is 2 bytes one way and
// 33/32 the other, some 6 VALU operations (T = 32768, four streams of C = 2048: pack
// 133 us, 6.1 TB/s, unpack 124, 6.5).
#include "elems.h"
#include "pack8.h"

namespace fmhc {

namespace {

// Lane i of a launch: row i / (4 G), group (i / 4) % G, quarter i % 4 of it.
// FLAT: C % 32 == 0, the tensor taken as one row (no division).  A launch
// covers at most 2^31 lanes.  A lane with fewer than 8 columns left takes the
// row's last 8, of which the first 8 - n are the lane's before (C >= 8).
struct Place {
  int64_t elem;   // first element of the lane's 8
  int64_t group;  // its scale byte
  int n;          // how many of the 8, the last ones, are this lane's (0 or less: none)
};
template <bool FLAT>
__device__ __forceinline__ Place place_of(uint32_t i, int C, uint32_t G) {
  const uint32_t grp = i >> 2, q = i & 3u;
  if constexpr (FLAT) {
    return Place{int64_t{i} * 8, grp, 8};
  } else {
    const uint32_t r = grp / G, g = grp - r * G;
    const int c = static_cast<int>(32u * g + 8u * q);
    return Place{int64_t{r} * C + (c < C - 8 ? c : C - 8), grp, C - c};
  }
}

// NT: the nontemporal hint, for whole aligned groups only: lines that two
// lanes' unaligned vectors share would be moved twice under it (T = 6007, C =
// 1001, four streams in fp32: pack 24 -> 20 us without, unpack 29 -> 20).
template <int DT, bool FLAT, bool NT>
__global__ __launch_bounds__(256) void pack8_kernel(const typename Elems<DT>::S* __restrict__ x,
                                                    int8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                    uint32_t lanes, int C, uint32_t G) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= lanes) return;  // whole quads
  const Place p = place_of<FLAT>(i, C, G);
  float f[8];
  Elems<DT>::template load8<NT>(x + p.elem, f);
  uint32_t m = 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __float_as_uint(f[e]) & 0x7fffffffu;
    m = (FLAT || e >= 8 - p.n) && b > m ? b : m;
  }
  const uint32_t E = pack_scale(quad_max(m));
  const u32x2 q = encode8(f, E);
  if (FLAT || p.n >= 8)
    st_codes<NT>(codes + p.elem, q);
  else if (p.n > 0)
    st_last_codes(codes + p.elem + 8 - p.n, q, p.n);
  if ((i & 3u) == 0) scales[p.group] = static_cast<uint8_t>(E);
}

// FLAT: a lane's 8 elements have one scale.
template <int DT, bool NT>
__global__ __launch_bounds__(256) void unpack8_kernel(const int8_t* __restrict__ codes,
                                                      const uint8_t* __restrict__ scales,
                                                      typename Elems<DT>::S* __restrict__ x, uint32_t lanes) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= lanes) return;
  float f[8];
  decode8(ld_codes<NT>(codes + int64_t{i} * 8), pack_unit(scales[i >> 2]), f);
  Elems<DT>::template store8<NT>(x + int64_t{i} * 8, f);
}

// Other widths, from 8 columns on: a lane takes 8 consecutive elements wherever
// rows begin and end, so that its load and its store are aligned as the tensors
// are (against 8 elements within a row: 10^6 rows of C = 65 in bf16 60 -> 44 us,
// 120044 of 1001 88 -> 83; with the nontemporal hint 80044 of 300 14 -> 18).  They
// are in at most two groups of their first element's row, and the first group of
// the next row.  A launch has at most 2^31 elements.
template <int DT>
__global__ __launch_bounds__(256) void unpack8_rows_kernel(const int8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ scales,
                                                           typename Elems<DT>::S* __restrict__ x, uint32_t n, uint32_t C,
                                                           uint32_t G) {
  const uint32_t chunk = blockIdx.x * 256u + threadIdx.x;
  if (chunk >= (n + 7u) / 8u) return;
  const uint32_t i = chunk * 8u;
  const uint32_t r = i / C, c = i - r * C;
  const uint32_t last = n - i < 8u ? n - i : 8u;       // elements of the chunk
  const uint32_t end = C - c < last ? C - c : last;    // those of row r
  const int64_t row = int64_t{r} * G;
  const float u0 = pack_unit(scales[row + (c >> 5)]);
  const float u1 = pack_unit(scales[row + ((c + end - 1u) >> 5)]);
  const float u2 = pack_unit(scales[end < last ? row + G : row]);
  const uint32_t n0 = kPackGroup - (c & (kPackGroup - 1));
  if (last == 8u) {
    float f[8];
    codes8(ld_codes<false>(codes + i), f);
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) f[e] *= e >= end ? u2 : e < n0 ? u0 : u1;
    Elems<DT>::template store8<false>(x + i, f);
  } else {
    for (uint32_t e = 0; e < last; ++e)
      Elems<DT>::store(x + i + e, static_cast<float>(codes[i + e]) * (e >= end ? u2 : e < n0 ? u0 : u1));
  }
}

// Rows of fewer than 8 columns, one lane each.
template <int DT>
__global__ __launch_bounds__(256) void pack8_short_kernel(const typename Elems<DT>::S* __restrict__ x,
                                                          int8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                          uint32_t rows, int C) {
  const uint32_t r = blockIdx.x * 256u + threadIdx.x;
  if (r >= rows) return;
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = e < C ? Elems<DT>::load(x + int64_t{r} * C + e) : 0.f;
  const uint32_t E = pack_scale(max_bits8(f));
  const u32x2 q = encode8(f, E);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < C) codes[int64_t{r} * C + e] = static_cast<int8_t>(q[e >> 2] >> (8 * (e & 3)));
  scales[r] = static_cast<uint8_t>(E);
}

template <int DT>
__global__ __launch_bounds__(256) void unpack8_short_kernel(const int8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales,
                                                            typename Elems<DT>::S* __restrict__ x, uint32_t rows, int C) {
  const uint32_t r = blockIdx.x * 256u + threadIdx.x;
  if (r >= rows) return;
  const float unit = pack_unit(scales[r]);
  for (int e = 0; e < C; ++e)
    Elems<DT>::store(x + int64_t{r} * C + e, static_cast<float>(codes[int64_t{r} * C + e]) * unit);
}

bool bad_sizes(int64_t rows, int64_t C) {
  return rows < 0 || C <= 0 || C > (int64_t{1} << 30) || rows > (int64_t{1} << 62) / (C + 32);
}

// f(first row, lanes) over pieces of at most 2^31 lanes (or elements), per_row for
// each row.
template <typename F>
void for_pieces(int64_t rows, int64_t per_row, F&& f) {
  const int64_t most = (int64_t{1} << 31) / per_row;  // C <= 2^30: at least 2
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    f(r, static_cast<uint32_t>(n * per_row));
  }
}

// lanes(flat, aligned) for rows of C columns from 8 on, few() below.
template <typename L, typename S>
int with_rows(int64_t C, bool aligned, L&& lanes, S&& few) {
  auto flat = [&](auto al) {
    C % kPackGroup == 0 ? lanes(std::true_type{}, al) : lanes(std::false_type{}, al);
  };
  if (C < 8)
    few();
  else
    aligned ? flat(std::true_type{}) : flat(std::false_type{});
  return launch_status();
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
    hipStream_t s = static_cast<hipStream_t>(stream);
    return with_rows(
        C, aligned16(x) && Pack8Src::aligned(codes),
        [&](auto flat, auto nt) {
          for_pieces(rows, 4 * int64_t{G}, [&](int64_t r, uint32_t lanes) {
            constexpr bool FLAT = decltype(flat)::value;
            pack8_kernel<DT, FLAT, FLAT && decltype(nt)::value><<<dim3(blocks_for(lanes, 256)), 256, 0, s>>>(
                xs + r * C, codes + r * C, scales + r * G, lanes, c, static_cast<uint32_t>(G));
          });
        },
        [&] {
          for_pieces(rows, 1, [&](int64_t r, uint32_t n) {
            pack8_short_kernel<DT><<<dim3(blocks_for(n, 256)), 256, 0, s>>>(xs + r * C, codes + r * C, scales + r, n, c);
          });
        });
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
    hipStream_t s = static_cast<hipStream_t>(stream);
    return with_rows(
        C, aligned16(x) && Pack8Src::aligned(codes),
        [&](auto flat, auto nt) {
          if constexpr (decltype(flat)::value) {
            for_pieces(rows, 4 * int64_t{G}, [&](int64_t r, uint32_t lanes) {
              unpack8_kernel<DT, decltype(nt)::value><<<dim3(blocks_for(lanes, 256)), 256, 0, s>>>(
                  codes + r * C, scales + r * G, xs + r * C, lanes);
            });
          } else {
            for_pieces(rows, C, [&](int64_t r, uint32_t n) {
              unpack8_rows_kernel<DT><<<dim3(blocks_for((int64_t{n} + 7) / 8, 256)), 256, 0, s>>>(
                  codes + r * C, scales + r * G, xs + r * C, n, static_cast<uint32_t>(c), static_cast<uint32_t>(G));
            });
          }
        },
        [&] {
          for_pieces(rows, 1, [&](int64_t r, uint32_t n) {
            unpack8_short_kernel<DT><<<dim3(blocks_for(n, 256)), 256, 0, s>>>(codes + r * C, scales + r, xs + r * C, n, c);
          });
        });
  });
}
