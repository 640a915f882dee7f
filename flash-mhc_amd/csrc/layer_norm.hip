// Layer norm over the last axis, forward and backward, with the input kept as
// it is or in 8 bits (pack8.h) for the backward.
//
//   forward   mean = sum_c x / C,  rstd = rsqrt(sum_c (x - mean)^2 / C + eps)
//             y = h w + b,  h = (x - mean) rstd
//   backward  g = gy w,  h = (x' - mean) rstd   (x' is x, or what its codes stand for)
//             grad_x = rstd (g - sum_c g / C - h sum_c g h / C)
//             grad_w = sum_t gy h,  grad_b = sum_t gy
//
// Everything is fp32 but the stored tensors, each rounded once.  A row is held
// in registers by LPT lanes, R groups of 8 columns each, so that the variance
// is taken around the mean (no difference of large sums) and x is read once;
// rows beyond that are read again from the caches.  In the backward a lane
// keeps the same columns for all rows of its workgroup and sums their grad_w and
// grad_b in registers; the workgroups' sums are added by a second kernel in a
// fixed order (no atomics: the results are deterministic).
#include <type_traits>

#include "elems.h"
#include "pack8.h"

namespace fmhc {

namespace {

constexpr int kLnBlock = 256;
constexpr int kLnWaves = kLnBlock / kWave;

// LPT lanes per row (a power of two up to one workgroup), R groups of 8 columns
// per lane; R = 0: rows of any length, read again for every use.  WHOLE: rows of
// whole, aligned groups, moved with the nontemporal hint.
template <int kLpt, int kRounds, bool kWhole>
struct LnWalk {
  static constexpr int LPT = kLpt, R = kRounds;
  static constexpr bool WHOLE = kWhole;
  static constexpr int SLOTS = kLnBlock / LPT;  // rows of a workgroup at a time
};

// The norm's weight and bias, in fp32 or x's type; either may be null (1, 0).
struct LnParams {
  const void* w;
  const void* b;
  bool f32;
};

template <int DT>
__device__ __forceinline__ void param8(const void* p, bool f32, int g, int n, float none, float (&f)[8]) {
  using S = typename Elems<DT>::S;
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = none;
  } else if (n >= 8) {
    if (f32)
      Elems<FMHC_DTYPE_F32>::load8<false>(static_cast<const float*>(p) + 8 * g, f);
    else
      Elems<DT>::template load8<false>(static_cast<const S*>(p) + 8 * g, f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      f[e] = e >= n ? 0.f
             : f32  ? static_cast<const float*>(p)[8 * g + e]
                    : Elems<DT>::load(static_cast<const S*>(p) + 8 * g + e);
  }
}

// Columns 8 g .. 8 g + 7 of a row of which n (any number) are inside; zeros
// beyond.
template <int DT, bool WHOLE>
__device__ __forceinline__ void row8(const typename Elems<DT>::S* row, int g, int n, float (&f)[8]) {
  if (WHOLE ? n > 0 : n >= 8) {
    Elems<DT>::template load8<WHOLE>(row + 8 * g, f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = !WHOLE && e < n ? Elems<DT>::load(row + 8 * g + e) : 0.f;
  }
}
template <int DT, bool WHOLE>
__device__ __forceinline__ void put8(typename Elems<DT>::S* row, int g, int n, const float (&f)[8]) {
  if (WHOLE ? n > 0 : n >= 8) {
    Elems<DT>::template store8<WHOLE>(row + 8 * g, f);
  } else if constexpr (!WHOLE) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) Elems<DT>::store(row + 8 * g + e, f[e]);
  }
}
template <bool WHOLE>
__device__ __forceinline__ void codes8(const int8_t* row, const uint8_t* scales, int g, int n, float (&f)[8]) {
  if (WHOLE ? n > 0 : n >= 8) {
    decode8(ld_codes<WHOLE>(row + 8 * g), pack_unit(scales[g >> 2]), f);
  } else {
    const float unit = !WHOLE && n > 0 ? pack_unit(scales[g >> 2]) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = !WHOLE && e < n ? static_cast<float>(row[8 * g + e]) * unit : 0.f;
  }
}

// The codes and the scale of the group of 32 columns whose quarter g this lane
// holds; the quad's four lanes are active.
template <bool WHOLE>
__device__ __forceinline__ void keep8(int8_t* row, uint8_t* scales, int g, int n, const float (&f)[8]) {
  const uint32_t E = pack_scale(quad_max(max_bits8(f)));
  const u32x2 q = encode8(f, E);
  if (WHOLE ? n > 0 : n >= 8) {
    st_codes<WHOLE>(row + 8 * g, q);
  } else if constexpr (!WHOLE) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) row[8 * g + e] = static_cast<int8_t>(q[e >> 2] >> (8 * (e & 3)));
  }
  if ((g & 3) == 0 && n > 0) scales[g >> 2] = static_cast<uint8_t>(E);
}

// Sum over a row's LPT lanes, in every one of them.  With several waves a row
// is a whole workgroup: the waves' sums are added in wave order through `red`,
// which the caller does not use again before another barrier.
template <int LPT>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (LPT <= kWave) {
    return group_sum<LPT>(v);
  } else {
    static_assert(LPT == kLnBlock, "a row is a whole workgroup");
    v = wave_sum(v);
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int w = 1; w < kLnWaves; ++w) s += red[w];
    return s;
  }
}

// f(g) for this lane's groups in a row of C columns; whole quads enter, so that
// lanes past the row's end take part with n <= 0.
template <typename WALK, typename F>
__device__ __forceinline__ void each_group(int sub, int C, F&& f) {
  const int ng = 4 * pack_groups(C);
  for (int g = sub; (g & ~3) < ng; g += WALK::LPT) f(g);
}

template <int DT, typename WALK, bool KEEP>
__global__ __launch_bounds__(kLnBlock) void ln_fwd_kernel(const typename Elems<DT>::S* __restrict__ x,
                                                          const LnParams P, typename Elems<DT>::S* __restrict__ y,
                                                          float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                          int8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                          int64_t T, int C, float eps) {
  constexpr int LPT = WALK::LPT, R = WALK::R;
  constexpr bool WHOLE = WALK::WHOLE;
  __shared__ float red[2][kLnWaves];
  const int sub = static_cast<int>(threadIdx.x) % LPT;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * WALK::SLOTS + static_cast<int>(threadIdx.x) / LPT;
  if (t >= T) return;  // a row's lanes leave together: no barrier is left waiting
  const auto* row = x + t * C;
  auto* out = y + t * C;
  int8_t* qrow = KEEP ? codes + t * C : nullptr;
  uint8_t* srow = KEEP ? scales + t * pack_groups(C) : nullptr;
  const float n_inv = 1.f / static_cast<float>(C);

  float v[R > 0 ? R : 1][8];
  float s = 0.f;
  if constexpr (R > 0) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      row8<DT, WHOLE>(row, sub + k * LPT, C - 8 * (sub + k * LPT), v[k]);
    }
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[k][e];
  } else {
    each_group<WALK>(sub, C, [&](int g) {
      row8<DT, WHOLE>(row, g, C - 8 * g, v[0]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[0][e];
    });
  }
  // Divided, not multiplied with 1 / C: the mean of equal values is that value.
  const float mean = row_sum<LPT>(s, red[0]) / static_cast<float>(C);

  float s2 = 0.f;
  auto spread = [&](const float (&f)[8], int n) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = f[e] - mean;
      s2 = (WHOLE ? n > 0 : e < n) ? __builtin_fmaf(d, d, s2) : s2;
    }
  };
  if constexpr (R > 0) {
#pragma unroll
    for (int k = 0; k < R; ++k) spread(v[k], C - 8 * (sub + k * LPT));
  } else {
    each_group<WALK>(sub, C, [&](int g) {
      row8<DT, WHOLE>(row, g, C - 8 * g, v[0]);
      spread(v[0], C - 8 * g);
    });
  }
  const float rstd = rsqrtf(row_sum<LPT>(s2, red[1]) * n_inv + eps);

  auto write = [&](const float (&f)[8], int g) __attribute__((always_inline)) {
    const int n = C - 8 * g;
    float w[8], b[8], o[8];
    param8<DT>(P.w, P.f32, g, n, 1.f, w);
    param8<DT>(P.b, P.f32, g, n, 0.f, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = __builtin_fmaf((f[e] - mean) * rstd, w[e], b[e]);
    put8<DT, WHOLE>(out, g, n, o);
    if constexpr (KEEP) keep8<WHOLE>(qrow, srow, g, n, f);
  };
  if constexpr (R > 0) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int g = sub + k * LPT;
      if ((g & ~3) < 4 * pack_groups(C)) write(v[k], g);
    }
  } else {
    each_group<WALK>(sub, C, [&](int g) {
      row8<DT, WHOLE>(row, g, C - 8 * g, v[0]);
      write(v[0], g);
    });
  }
  if (sub == 0) {
    if (mean_out) mean_out[t] = mean;
    if (rstd_out) rstd_out[t] = rstd;
  }
}

// Rows t, t + step, ... of a workgroup.  partial (may be null): this
// workgroup's sums, [2][cols] with cols = 8 ceil(C / 8): grad_w, then grad_b.
// SRC: x in DT, or its codes and scales.
template <int DT, typename WALK, bool KEPT>
__global__ __launch_bounds__(kLnBlock) void ln_bwd_kernel(
    const typename Elems<DT>::S* __restrict__ gy, const std::conditional_t<KEPT, int8_t, typename Elems<DT>::S>* __restrict__ x,
    const uint8_t* __restrict__ scales, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
    const LnParams P, typename Elems<DT>::S* __restrict__ gx, float* __restrict__ partial, int64_t T, int C) {
  constexpr int LPT = WALK::LPT, R = WALK::R, SLOTS = WALK::SLOTS;
  constexpr bool WHOLE = WALK::WHOLE;
  __shared__ float red[2][2][kLnWaves];
  const int sub = static_cast<int>(threadIdx.x) % LPT;
  const int slot = static_cast<int>(threadIdx.x) / LPT;
  const int64_t step = static_cast<int64_t>(gridDim.x) * SLOTS;
  const float n_inv = 1.f / static_cast<float>(C);
  const int G = pack_groups(C);

  constexpr int RR = R > 0 ? R : 1;
  float w[RR][8], dw[RR][8], db[RR][8];
#pragma unroll
  for (int k = 0; k < RR; ++k) {
    if constexpr (R > 0) param8<DT>(P.w, P.f32, sub + k * LPT, C - 8 * (sub + k * LPT), 1.f, w[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[k][e] = db[k][e] = 0.f;
  }

  int parity = 0;
  // Every wave of the workgroup walks as many rows where a row has a barrier
  // (SLOTS = 1 then).
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * SLOTS + slot; t < T; t += step) {
    const auto* grow = gy + t * C;
    const auto* xrow = x + t * C;
    const uint8_t* srow = KEPT ? scales + t * G : nullptr;
    auto* orow = gx + t * C;
    const float mean = mean_in[t], rstd = rstd_in[t];
    auto fetch = [&](int g, float (&q)[8], float (&h)[8]) __attribute__((always_inline)) {
      const int n = C - 8 * g;
      row8<DT, WHOLE>(grow, g, n, q);
      if constexpr (KEPT)
        codes8<WHOLE>(xrow, srow, g, n, h);
      else
        row8<DT, WHOLE>(xrow, g, n, h);
    };
    // Columns past the row's end have gy = 0, and so add nothing to any sum.
    float q[RR][8], h[RR][8], s1 = 0.f, s2 = 0.f;
    auto sums = [&](const float (&qk)[8], float (&hk)[8], const float (&wk)[8]) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        hk[e] = (hk[e] - mean) * rstd;
        const float g = qk[e] * wk[e];
        s1 += g;
        s2 = __builtin_fmaf(g, hk[e], s2);
      }
    };
    if constexpr (R > 0) {
#pragma unroll
      for (int k = 0; k < R; ++k) fetch(sub + k * LPT, q[k], h[k]);
#pragma unroll
      for (int k = 0; k < R; ++k) sums(q[k], h[k], w[k]);
    } else {
      each_group<WALK>(sub, C, [&](int g) {
        fetch(g, q[0], h[0]);
        param8<DT>(P.w, P.f32, g, C - 8 * g, 1.f, w[0]);
        sums(q[0], h[0], w[0]);
      });
    }
    if constexpr (LPT <= kWave) {
      s1 = group_sum<LPT>(s1);
      s2 = group_sum<LPT>(s2);
    } else {
      // One barrier a row: the next row's sums go to the other half, and a wave
      // writes this half again only behind the next row's barrier.
      s1 = wave_sum(s1);
      s2 = wave_sum(s2);
      if ((threadIdx.x & (kWave - 1)) == 0) {
        red[parity][0][threadIdx.x >> 6] = s1;
        red[parity][1][threadIdx.x >> 6] = s2;
      }
      __syncthreads();
      s1 = red[parity][0][0];
      s2 = red[parity][1][0];
#pragma unroll
      for (int i = 1; i < kLnWaves; ++i) {
        s1 += red[parity][0][i];
        s2 += red[parity][1][i];
      }
      parity ^= 1;
    }
    const float c1 = s1 * n_inv, c2 = s2 * n_inv;
    auto write = [&](int g, const float (&qk)[8], const float (&hk)[8], const float (&wk)[8]) __attribute__((always_inline)) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = rstd * (qk[e] * wk[e] - c1 - hk[e] * c2);
      put8<DT, WHOLE>(orow, g, C - 8 * g, o);
    };
    if constexpr (R > 0) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        write(sub + k * LPT, q[k], h[k], w[k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dw[k][e] = __builtin_fmaf(q[k][e], h[k][e], dw[k][e]);
          db[k][e] += q[k][e];
        }
      }
    } else {
      each_group<WALK>(sub, C, [&](int g) {
        fetch(g, q[0], h[0]);
        param8<DT>(P.w, P.f32, g, C - 8 * g, 1.f, w[0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[0][e] = (h[0][e] - mean) * rstd;
        write(g, q[0], h[0], w[0]);
      });
    }
  }
  if constexpr (R > 0) {
    if (!partial) return;
    const int cols = (C + 7) / 8 * 8;
    float* dst = partial + static_cast<int64_t>(blockIdx.x) * 2 * cols;
    if constexpr (SLOTS == 1) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int c = 8 * (sub + k * LPT);
        if (c < cols) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            dst[c + e] = dw[k][e];
            dst[cols + c + e] = db[k][e];
          }
        }
      }
    } else {
      // The rows that one wave holds side by side, then the waves in order.
      constexpr int kCols = LPT < kWave ? 8 * LPT : 8 * LPT * R;  // of a wave
      __shared__ float acc[2][kCols];
      static_assert(LPT >= kWave || R == 1, "several rows per wave hold one group per lane");
      const int wave = static_cast<int>(threadIdx.x) >> 6;
      const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
      for (int k = 0; k < R; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int m = LPT; m < kWave; m <<= 1) {
            dw[k][e] += __shfl_xor(dw[k][e], m, kWave);
            db[k][e] += __shfl_xor(db[k][e], m, kWave);
          }
      for (int i = 0; i < kLnWaves; ++i) {
        if (wave == i && lane < LPT) {
#pragma unroll
          for (int k = 0; k < R; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int at = (k * 8 + e) * (LPT < kWave ? LPT : kWave) + sub;
              acc[0][at] = i == 0 ? dw[k][e] : acc[0][at] + dw[k][e];
              acc[1][at] = i == 0 ? db[k][e] : acc[1][at] + db[k][e];
            }
        }
        __syncthreads();
      }
      for (int c = static_cast<int>(threadIdx.x); c < cols; c += kLnBlock) {
        const int g = c / 8, at = (g / LPT * 8 + c % 8) * LPT + g % LPT;
        dst[c] = acc[0][at];
        dst[cols + c] = acc[1][at];
      }
    }
  }
}

// grad_w and grad_b of rows too long for registers: a workgroup takes 256
// columns and rows blockIdx.y, blockIdx.y + gridDim.y, ..., into `partial` as
// ln_bwd_kernel's workgroup blockIdx.y.
template <int DT, bool KEPT>
__global__ __launch_bounds__(kLnBlock) void ln_columns_kernel(
    const typename Elems<DT>::S* __restrict__ gy, const std::conditional_t<KEPT, int8_t, typename Elems<DT>::S>* __restrict__ x,
    const uint8_t* __restrict__ scales, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
    float* __restrict__ partial, int64_t T, int C) {
  const int cols = (C + 7) / 8 * 8;
  const int c = static_cast<int>(blockIdx.x) * kLnBlock + static_cast<int>(threadIdx.x);
  if (c >= cols) return;
  float dw = 0.f, db = 0.f;
  if (c < C) {
    for (int64_t t = blockIdx.y; t < T; t += gridDim.y) {
      const float q = Elems<DT>::load(gy + t * C + c);
      float v;
      if constexpr (KEPT)
        v = static_cast<float>(x[t * C + c]) * pack_unit(scales[t * pack_groups(C) + (c >> 5)]);
      else
        v = Elems<DT>::load(x + t * C + c);
      dw = __builtin_fmaf(q, (v - mean_in[t]) * rstd_in[t], dw);
      db += q;
    }
  }
  float* dst = partial + static_cast<int64_t>(blockIdx.y) * 2 * cols;
  dst[c] = dw;
  dst[cols + c] = db;
}

// grad_w and grad_b from the workgroups' sums: 16 columns of four per workgroup,
// 16 shares of the rows, added in order.
template <int DT>
__global__ __launch_bounds__(kLnBlock) void ln_reduce_kernel(const float* __restrict__ partial, int64_t parts,
                                                             int cols, int C, bool f32, void* __restrict__ gw,
                                                             void* __restrict__ gb) {
  constexpr int kVecs = 16, kShares = kLnBlock / kVecs;
  __shared__ f32x4 acc[kShares][kVecs];
  const int v = static_cast<int>(threadIdx.x) % kVecs, share = static_cast<int>(threadIdx.x) / kVecs;
  const int i = (static_cast<int>(blockIdx.x) * kVecs + v) * 4;  // of 2 cols, a multiple of 16
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (i < 2 * cols) {
    const float* src = partial + i;
#pragma unroll 4
    for (int64_t p = share; p < parts; p += kShares) s += *reinterpret_cast<const f32x4*>(src + p * 2 * cols);
  }
  acc[share][v] = s;
  __syncthreads();
  if (share != 0 || i >= 2 * cols) return;
#pragma unroll
  for (int k = 1; k < kShares; ++k) s += acc[k][v];
  void* dst = i < cols ? gw : gb;
  if (!dst) return;
  const int c = i < cols ? i : i - cols;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (c + e < C) {
      if (f32)
        static_cast<float*>(dst)[c + e] = s[e];
      else
        Elems<DT>::store(static_cast<typename Elems<DT>::S*>(dst) + c + e, s[e]);
    }
  }
}

// Zero gradients of the parameters of an empty batch (a kernel, not a memset,
// so that the call can be captured in a graph).
__global__ __launch_bounds__(kLnBlock) void ln_zero_kernel(uint16_t* __restrict__ p, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kLnBlock + threadIdx.x;
  if (i < n) p[i] = 0;
}

// f(LnWalk) for rows of C columns.
template <typename F>
void with_ln_walk(int C, bool whole, F&& f) {
  auto pick = [&](auto wh) {
    constexpr bool W = decltype(wh)::value;
    if (C <= 64) return f(LnWalk<8, 1, W>{});
    if (C <= 128) return f(LnWalk<16, 1, W>{});
    if (C <= 256) return f(LnWalk<32, 1, W>{});
    if (C <= 512) return f(LnWalk<64, 1, W>{});
    if (C <= 1024) return f(LnWalk<64, 2, W>{});
    if (C <= 2048) return f(LnWalk<256, 1, W>{});
    if (C <= 4096) return f(LnWalk<256, 2, W>{});
    if (C <= 8192) return f(LnWalk<256, 4, W>{});
    if (C <= 16384) return f(LnWalk<256, 8, W>{});
    return f(LnWalk<256, 0, W>{});
  };
  whole ? pick(std::true_type{}) : pick(std::false_type{});
}

// Rows of a workgroup of the backward at a time.
int ln_slots(int C) {
  int n = 1;
  with_ln_walk(C, true, [&](auto w) { n = decltype(w)::SLOTS; });
  return n;
}

// Workgroups of the backward, whose sums the reduce adds.
constexpr int64_t kLnParts = 1024;
int64_t ln_parts(int64_t T, int C) {
  const int64_t slots = ln_slots(C);
  const int64_t n = (T + slots - 1) / slots;
  return n < kLnParts ? n : kLnParts;
}

int64_t ln_workspace(int64_t T, int64_t C) {
  return ln_parts(T, static_cast<int>(C)) * 2 * ((C + 7) / 8 * 8) * static_cast<int64_t>(sizeof(float));
}

bool bad_sizes(int64_t T, int64_t C) {
  return T < 0 || C <= 0 || C > (int64_t{1} << 28) || T > (int64_t{1} << 60) / C;
}

// Element sizes of the two types; the parameters are fp32 or of x's type.
bool bad_types(int dtype, int param_dtype) {
  if (dtype != FMHC_DTYPE_F32 && dtype != FMHC_DTYPE_BF16 && dtype != FMHC_DTYPE_F16) return true;
  return param_dtype != FMHC_DTYPE_F32 && param_dtype != dtype;
}

}  // namespace
}  // namespace fmhc

extern "C" int fmhc_layer_norm_fwd(const void* x, const void* weight, const void* bias, void* y, float* mean,
                                   float* rstd, int8_t* x_codes, uint8_t* x_scales, int dtype, int param_dtype,
                                   int64_t T, int64_t C, float eps, void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C) || bad_types(dtype, param_dtype) || !x_codes != !x_scales) return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (!x || !y) return FMHC_ERR_INVALID_ARGUMENT;
  return with_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    using S = typename Elems<DT>::S;
    const auto* xs = static_cast<const S*>(x);
    auto* ys = static_cast<S*>(y);
    const int c = static_cast<int>(C), G = pack_groups(c);
    const LnParams P{weight, bias, param_dtype == FMHC_DTYPE_F32};
    const bool whole = C % 8 == 0 && aligned16(x) && aligned16(y) && (!x_codes || Pack8Src::aligned(x_codes));
    with_ln_walk(c, whole, [&](auto w) {
      using Walk = decltype(w);
      for_launches(T, kLnBlock, Walk::SLOTS, [&](int64_t t, int64_t n) {
        auto launch = [&](auto keep) {
          constexpr bool KEEP = decltype(keep)::value;
          ln_fwd_kernel<DT, Walk, KEEP><<<dim3(blocks_for(n, Walk::SLOTS)), kLnBlock, 0, static_cast<hipStream_t>(stream)>>>(
              xs + t * C, P, ys + t * C, mean ? mean + t : nullptr, rstd ? rstd + t : nullptr,
              KEEP ? x_codes + t * C : nullptr, KEEP ? x_scales + t * G : nullptr, n, c, eps);
        };
        x_codes ? launch(std::true_type{}) : launch(std::false_type{});
      });
    });
    return launch_status();
  });
}

extern "C" int64_t fmhc_layer_norm_bwd_workspace_bytes(int64_t T, int64_t C) {
  if (fmhc::bad_sizes(T, C) || T == 0) return 0;
  return fmhc::ln_workspace(T, C);
}

namespace {

template <int DT, bool KEPT, typename X>
int ln_bwd_run(const void* grad_y, const X* xs, const uint8_t* scales, const float* mean, const float* rstd,
               const void* weight, void* grad_x, void* grad_w, void* grad_b, void* workspace, bool f32, int64_t T,
               int64_t C, hipStream_t s) {
  using namespace fmhc;
  using S = typename Elems<DT>::S;
  const auto* gy = static_cast<const S*>(grad_y);
  auto* gx = static_cast<S*>(grad_x);
  const int c = static_cast<int>(C);
  const bool whole = C % 8 == 0 && aligned16(gy) && aligned16(gx) && ((reinterpret_cast<uintptr_t>(xs) & (KEPT ? 7u : 15u)) == 0);
  const int64_t parts = ln_parts(T, c);
  float* partial = grad_w || grad_b ? static_cast<float*>(workspace) : nullptr;
  const LnParams P{weight, nullptr, f32};
  with_ln_walk(c, whole, [&](auto w) {
    using Walk = decltype(w);
    ln_bwd_kernel<DT, Walk, KEPT><<<dim3(static_cast<unsigned>(parts)), kLnBlock, 0, s>>>(gy, xs, scales, mean, rstd, P,
                                                                                         gx, partial, T, c);
    if (Walk::R == 0 && partial)
      ln_columns_kernel<DT, KEPT><<<dim3(blocks_for((C + 7) / 8 * 8, kLnBlock), static_cast<unsigned>(parts)), kLnBlock, 0,
                                    s>>>(gy, xs, scales, mean, rstd, partial, T, c);
  });
  const int st = launch_status();
  if (st != FMHC_OK || !partial) return st;
  const int cols = (c + 7) / 8 * 8;
  ln_reduce_kernel<DT><<<dim3(blocks_for(2 * static_cast<int64_t>(cols), 64)), kLnBlock, 0, s>>>(partial, parts, cols, c,
                                                                                               f32, grad_w, grad_b);
  return launch_status();
}

}  // namespace

extern "C" int fmhc_layer_norm_bwd(const void* grad_y, const void* x, const int8_t* x_codes, const uint8_t* x_scales,
                                   const float* mean, const float* rstd, const void* weight, void* grad_x,
                                   void* grad_weight, void* grad_bias, void* workspace, int64_t workspace_bytes,
                                   int dtype, int param_dtype, int64_t T, int64_t C, void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C) || bad_types(dtype, param_dtype) || !x_codes != !x_scales || (x && x_codes))
    return FMHC_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f32 = param_dtype == FMHC_DTYPE_F32;
  if (T == 0) {
    const int64_t n = C * (f32 ? 2 : 1);  // 16-bit words of a parameter's gradient
    for (void* p : {grad_weight, grad_bias})
      if (p) ln_zero_kernel<<<dim3(blocks_for(n, kLnBlock)), kLnBlock, 0, s>>>(static_cast<uint16_t*>(p), n);
    return launch_status();
  }
  if (!grad_y || (!x && !x_codes) || !mean || !rstd || !grad_x) return FMHC_ERR_INVALID_ARGUMENT;
  if ((grad_weight || grad_bias) && (!workspace || workspace_bytes < ln_workspace(T, C) || !aligned16(workspace)))
    return FMHC_ERR_INVALID_ARGUMENT;
  return with_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    using S = typename Elems<DT>::S;
    return x_codes ? ln_bwd_run<DT, true>(grad_y, x_codes, x_scales, mean, rstd, weight, grad_x, grad_weight, grad_bias,
                                          workspace, f32, T, C, s)
                   : ln_bwd_run<DT, false>(grad_y, static_cast<const S*>(x), nullptr, mean, rstd, weight, grad_x,
                                           grad_weight, grad_bias, workspace, f32, T, C, s);
  });
}
