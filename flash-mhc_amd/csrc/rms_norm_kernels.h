// The RMS norm's kernels, for the translation unit of one storage type.
//
// Rows lie over lanes as the layer norm's do (layer_norm_kernels.h): LPT lanes hold
// a row, R groups of 8 columns each, from its loads to its stores, a lane keeps the
// same columns for every row of its workgroup, and the next row's loads are issued
// before the current row is computed.  One pass: the sum of squares needs no mean,
// and a packed row's maximum is that of |s w|, whose product with rstd is the norm's.
// Bound by HBM, in bf16: T = 65536, C = 2048 with a residual (8 bytes an element) the
// forward takes 172 us (6.2 TB/s), the backward 167 + 4.8 for the weight's sums (6.4);
// without one 88 and 129; T = 65536, C = 1024 in 8 bits 34 to 36 (3 bytes an element,
// 5.6 to 5.9 TB/s).  One row of 4096: 2.5 us, a launch's latency.
#pragma once

#include "layer_norm_kernels.h"
#include "rms_norm.h"

namespace fmhc {

namespace {

// The maximum over the LPT consecutive lanes of a row, in every one of them.
template <int LPT>
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
#pragma unroll
  for (int k = (LPT < kWave ? LPT : kWave) / 2; k >= 1; k >>= 1) {
    const uint32_t o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), k, kWave));
    m = o > m ? o : m;
  }
  return m;
}

// A row's sum and (MAX) maximum over its LPT lanes of a workgroup of BLOCK threads, in
// every lane; halves of `red` in turn, as LnSums.
template <int LPT, int BLOCK, bool MAX>
struct RmsStats {
  static constexpr int WPR = LPT > kWave ? LPT / kWave : 1;
  uint32_t (*red)[BLOCK / kWave][2];  // [2]
  int half = 0;
  __device__ __forceinline__ void operator()(float& s, uint32_t& m) {
    if constexpr (WPR == 1) {
      s = group_sum<LPT>(s);
      if constexpr (MAX) m = group_max<LPT>(m);
    } else {
      const int wave = static_cast<int>(threadIdx.x) >> 6;
      s = wave_sum(s);
      if constexpr (MAX) m = group_max<kWave>(m);
      if ((threadIdx.x & (kWave - 1)) == 0) {
        red[half][wave][0] = __float_as_uint(s);
        if constexpr (MAX) red[half][wave][1] = m;
      }
      __syncthreads();
      const int first = wave & ~(WPR - 1);
      s = __uint_as_float(red[half][first][0]);
      if constexpr (MAX) m = red[half][first][1];
#pragma unroll
      for (int w = 1; w < WPR; ++w) {
        s += __uint_as_float(red[half][first + w][0]);
        if constexpr (MAX) {
          const uint32_t o = red[half][first + w][1];
          m = o > m ? o : m;
        }
      }
      half ^= 1;
    }
  }
};

// A packed row's scale and the factor of its codes, from the bits of its largest magnitude
// before rstd: code = round_half_even(v 127 / top), scale = top / 127.  Inf or NaN in the row:
// scale NaN, codes 0.  A magnitude below the normal numbers has too few bits for a scale where
// rstd is large (eps near 0): such a row counts as zero.
struct RowScale {
  float scale, to_code;
  uint32_t keep;
};
__device__ __forceinline__ RowScale row_scale(uint32_t m, float rstd) {
  float top = __uint_as_float(m) * rstd;
  const bool finite = top < __builtin_inff(), some = finite && m >= 0x00800000u;
  top = some ? fmaxf(top, kRowLeast) : kRowLeast;
  return RowScale{finite ? top / 127.f : __uint_as_float(0x7fc00000u), some ? 127.f / top : 0.f, some ? ~0u : 0u};
}

// v 127 / top is rounded, so that half the largest magnitude (a common value in 16 bits) is 63.5
// and not beside it; the addition of 1.5 x 2^23 then rounds half to even and leaves the code in the
// sum's low byte.  |v| to_code is at most 127 (1 + 2^-22).
__device__ __forceinline__ uint32_t row_code(float v, float to_code) {
#pragma clang fp contract(off)
  return __float_as_uint(v * to_code + 12582912.f);
}

__device__ __forceinline__ u32x2 row_codes8(const float (&v)[8], const RowScale& r) {
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = row_code(v[e], r.to_code);
  u32x2 q;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x0c0c0400u);
    q[h] = (lo | hi << 16) & r.keep;
  }
  return q;
}

// What the forward leaves of a row.
constexpr int kRmsY = 0;      // the norm in x's type
constexpr int kRmsCodes = 1;  // the norm's codes, from its fp32 values
constexpr int kRmsRows = 2;   // the codes of the row itself

template <int DT, int LPT, int R, bool NT, bool ADD, int OUT>
__global__ __launch_bounds__(ln_fwd_block<LPT>()) void rms_fwd_kernel(
    const typename Elems<DT>::S* __restrict__ x, const typename Elems<DT>::S* __restrict__ r,
    const void* __restrict__ wp, bool w_f32, typename Elems<DT>::S* __restrict__ y, int8_t* __restrict__ codes,
    float* __restrict__ scales, int64_t ld_codes, typename Elems<DT>::S* __restrict__ sum,
    float* __restrict__ rstd_out, int64_t T, int C, float eps) {
  constexpr int BLOCK = ln_fwd_block<LPT>(), SLOTS = BLOCK / LPT;
  __shared__ uint32_t red[2][BLOCK / kWave][2];
  RmsStats<LPT, BLOCK, OUT != kRmsY> stats{red};
  const int sub = static_cast<int>(threadIdx.x) % LPT, slot = static_cast<int>(threadIdx.x) / LPT;
  const float n_inv = 1.f / static_cast<float>(C);

  LnPlace at[R];
  float w[R][8];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    at[k] = ln_place(sub + k * LPT, C);
    if constexpr (OUT != kRmsRows) ln_param8<DT>(wp, w_f32, at[k].c, 1.f, w[k]);
  }
  // Only a lane's last group can be short or past the row's end.
  auto inside = [&](int k, int e) { return k < R - 1 || e >= at[k].skip; };

  // Every thread walks as many rows (the barriers of RmsStats), those past the
  // last one on the last one's data, without storing.
  const int64_t step = static_cast<int64_t>(gridDim.x) * SLOTS;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * SLOTS;
  LnRaw<DT> raw[R], rawr[ADD ? R : 1];
  auto load = [&](int64_t t) {
    const int64_t at0 = (t < T ? t : T - 1) * C;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      raw[k] = ln_load<DT, NT>(x + at0 + at[k].c);
      if constexpr (ADD) rawr[k] = ln_load<DT, NT>(r + at0 + at[k].c);
    }
  };
  load(first + slot);
  for (int64_t t0 = first; t0 < T; t0 += step) {
    const int64_t t = t0 + slot;
    float v[R][8];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      ln_unpack<DT>(raw[k], v[k]);
      if constexpr (ADD) {
        float f[8];
        ln_unpack<DT>(rawr[k], f);
        // The norm is that of the sum as it is kept.
#pragma unroll
        for (int e = 0; e < 8; ++e) v[k][e] = Elems<DT>::rounded(v[k][e] + f[e]);
      }
    }
    if (t0 + step < T) load(t + step);
    __builtin_amdgcn_sched_barrier(0);

    float s = 0.f, rstd = 1.f;
    uint32_t m = 0u;
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = inside(k, e) ? v[k][e] : 0.f;
        if constexpr (OUT != kRmsRows) s = __builtin_fmaf(d, d, s);
        if constexpr (OUT != kRmsY) {
          // (A column that is held twice changes no maximum.)
          const float vw = OUT == kRmsRows ? v[k][e] : v[k][e] * w[k][e];
          const uint32_t bits = __float_as_uint(vw) & 0x7fffffffu;
          m = bits > m ? bits : m;
        }
      }
    stats(s, m);
    if constexpr (OUT != kRmsRows) rstd = rsqrtf(s * n_inv + eps);
    RowScale rs;
    if constexpr (OUT != kRmsY) rs = row_scale(m, rstd);
    if (t < T) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (k == R - 1 && at[k].skip == 8) continue;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = OUT == kRmsRows ? v[k][e] : v[k][e] * rstd * w[k][e];
        if constexpr (OUT == kRmsY)
          Elems<DT>::template store8<NT>(y + t * C + at[k].c, o);
        else
          st_codes<NT>(codes + t * ld_codes + at[k].c, row_codes8(o, rs));
        if constexpr (ADD) Elems<DT>::template store8<NT>(sum + t * C + at[k].c, v[k]);
      }
      if (sub == 0) {
        if constexpr (OUT == kRmsY) {
          if (rstd_out) rstd_out[t] = rstd;
        } else {
          scales[t] = rs.scale;
        }
      }
    }
  }
}

// grad_w of kRmsColumns columns from `group` kRmsColumns on, from all rows: it needs no row's sum.
constexpr int kRmsColumns = 64;
constexpr int kRmsPitch = kLnBwdBlock + 4;
template <int DT>
__device__ __forceinline__ void rms_columns(const typename Elems<DT>::S* __restrict__ gy,
                                            const typename Elems<DT>::S* __restrict__ x,
                                            const float* __restrict__ rstd_in, bool w_f32, void* __restrict__ gw,
                                            float* acc, int group, int64_t T, int C) {
  constexpr int BLOCK = kLnBwdBlock, VECS = kRmsColumns / 8, SLOTS = BLOCK / VECS;
  const int own = static_cast<int>(threadIdx.x) % VECS, slot = static_cast<int>(threadIdx.x) / VECS;
  const LnPlace p = ln_place(group * VECS + own, C);
  float dw[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[e] = 0.f;
#pragma unroll 4
  for (int64_t t = slot; t < T; t += SLOTS) {
    float q[8], h[8];
    ln_unpack<DT>(ln_load<DT, false>(gy + t * C + p.c), q);
    ln_unpack<DT>(ln_load<DT, false>(x + t * C + p.c), h);
    const float rstd = rstd_in[t];
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[e] = __builtin_fmaf(q[e], h[e] * rstd, dw[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e * kRmsPitch + threadIdx.x] = dw[e];
  __syncthreads();
  // A column's slots: eight threads add eight each, one adds their sums.
  constexpr int SHARE = SLOTS / 8;
  const int c = static_cast<int>(threadIdx.x) % kRmsColumns, part = static_cast<int>(threadIdx.x) / kRmsColumns;
  const float* src = acc + c % 8 * kRmsPitch + c / 8;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < SHARE; ++k) s += src[(part * SHARE + k) * VECS];
  __syncthreads();
  acc[part * kRmsColumns + c] = s;
  __syncthreads();
  if (part != 0) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += acc[k * kRmsColumns + c];
  const LnPlace at = ln_place(group * VECS + c / 8, C);
  if (c % 8 < at.skip) return;
  const int64_t n = at.c + c % 8;
  if (w_f32)
    static_cast<float*>(gw)[n] = s;
  else
    Elems<DT>::store(static_cast<typename Elems<DT>::S*>(gw) + n, s);
}

// partial (may be null): this workgroup's sums of grad_w, rms_cols(C) of them.  The first col_groups
// workgroups take columns of grad_w instead of rows (then partial is null).
template <int DT, int LPT, int R, bool NT, bool GI>
__global__ __launch_bounds__(kLnBwdBlock) void rms_bwd_kernel(
    const typename Elems<DT>::S* __restrict__ gy, const typename Elems<DT>::S* __restrict__ x,
    const float* __restrict__ rstd_in, const void* __restrict__ wp, bool w_f32,
    const typename Elems<DT>::S* __restrict__ gi, typename Elems<DT>::S* __restrict__ gx, float* __restrict__ partial,
    void* __restrict__ gw, int col_groups, int64_t T, int C) {
  constexpr int BLOCK = kLnBwdBlock, SLOTS = BLOCK / LPT;
  __shared__ float red[2][BLOCK / kWave][1];
  __shared__ float acc[8 * kRmsPitch];
  if (static_cast<int>(blockIdx.x) < col_groups)
    return rms_columns<DT>(gy, x, rstd_in, w_f32, gw, acc, static_cast<int>(blockIdx.x), T, C);
  const int64_t group = static_cast<int>(blockIdx.x) - col_groups, groups = static_cast<int>(gridDim.x) - col_groups;
  LnSums<LPT, BLOCK, 1> row_sum{red};
  const int sub = static_cast<int>(threadIdx.x) % LPT, slot = static_cast<int>(threadIdx.x) / LPT;
  const float n_inv = 1.f / static_cast<float>(C);

  LnPlace at[R];
  float w[R][8], dw[R][8];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    at[k] = ln_place(sub + k * LPT, C);
    ln_param8<DT>(wp, w_f32, at[k].c, 1.f, w[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[k][e] = 0.f;
  }

  const int64_t step = groups * SLOTS;
  const int64_t first = group * SLOTS;
  LnRaw<DT> rg[R], rx[R], ri[GI ? R : 1];
  float rstd_n;
  auto load = [&](int64_t tt) {
    const int64_t t = tt < T ? tt : T - 1;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      rg[k] = ln_load<DT, NT>(gy + t * C + at[k].c);
      rx[k] = ln_load<DT, NT>(x + t * C + at[k].c);
      if constexpr (GI) ri[k] = ln_load<DT, NT>(gi + t * C + at[k].c);
    }
    rstd_n = rstd_in[t];
  };
  load(first + slot);
  for (int64_t t0 = first; t0 < T; t0 += step) {
    const int64_t t = t0 + slot;
    const float rstd = rstd_n;
    // Few groups per lane stay in fp32 between the sum and the stores; more stay as
    // loaded and are widened again.
    constexpr bool HOLD = R <= 3;
    LnRaw<DT> cg[R], cx[R], ci[GI ? R : 1];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      cg[k] = rg[k];
      cx[k] = rx[k];
      if constexpr (GI) ci[k] = ri[k];
    }
    if (t0 + step < T) load(t + step);
    __builtin_amdgcn_sched_barrier(0);
    float q[HOLD ? R : 1][8], h[HOLD ? R : 1][8];
    auto widen = [&](int k, float (&qk)[8], float (&hk)[8]) __attribute__((always_inline)) {
      ln_unpack<DT>(cg[k], qk);
      ln_unpack<DT>(cx[k], hk);
#pragma unroll
      for (int e = 0; e < 8; ++e) hk[e] *= rstd;
    };

    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float (&qk)[8] = q[HOLD ? k : 0];
      float (&hk)[8] = h[HOLD ? k : 0];
      widen(k, qk, hk);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float g = k < R - 1 || e >= at[k].skip ? qk[e] * w[k][e] : 0.f;
        s[0] = __builtin_fmaf(g, hk[e], s[0]);
      }
    }
    row_sum(s);
    if constexpr (!HOLD) {
      // The compiler is not to keep the widened values after all.
#pragma unroll
      for (int k = 0; k < R; ++k) {
        ln_opaque(cg[k]);
        ln_opaque(cx[k]);
      }
    }
    if (t < T) {
      const float c2 = s[0] * n_inv * rstd;
      auto* out = gx + t * C;
#pragma unroll
      for (int k = 0; k < R; ++k) {
        float (&qk)[8] = q[HOLD ? k : 0];
        float (&hk)[8] = h[HOLD ? k : 0];
        if constexpr (!HOLD) widen(k, qk, hk);
        float o[8], f[8];
        if constexpr (GI) ln_unpack<DT>(ci[k], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // rstd (g - h sum(g h) / C), and x's other gradient, rounded once.
          o[e] = __builtin_fmaf(qk[e] * w[k][e], rstd, -hk[e] * c2);
          if constexpr (GI) o[e] += f[e];
          dw[k][e] = __builtin_fmaf(qk[e], hk[e], dw[k][e]);
        }
        if (k < R - 1 || at[k].skip < 8) Elems<DT>::template store8<NT>(out + at[k].c, o);
      }
    }
  }
  if (!partial) return;
  // The workgroup's rows: the threads that hold the same columns, in slot order.
  float* dst = partial + static_cast<int64_t>(blockIdx.x) * ((C + 7) / 8 * 8);
#pragma unroll
  for (int k = 0; k < R; ++k) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e * kRmsPitch + threadIdx.x] = dw[k][e];
    __syncthreads();
    for (int i = static_cast<int>(threadIdx.x); i < 8 * LPT; i += BLOCK) {
      const int own = i / 8, e = i % 8;
      const float* src = acc + e * kRmsPitch + own;
      float v = src[0];
#pragma unroll
      for (int sl = 1; sl < SLOTS; ++sl) v += src[sl * LPT];
      const LnPlace p = ln_place(own + k * LPT, C);
      if (e >= p.skip) dst[p.c + e] = v;
    }
  }
}

// ---------------------------------------------------------------------------
// Rows of fewer than 8 columns and rows that no registers hold, as the layer
// norm's: one workgroup per row, which is read again for every use, from L2.

template <int DT, int N, int OUT>
__global__ __launch_bounds__(ln_any_block<N>()) void rms_fwd_any(
    const typename Elems<DT>::S* __restrict__ x, const typename Elems<DT>::S* __restrict__ r,
    const void* __restrict__ wp, bool w_f32, typename Elems<DT>::S* __restrict__ y, int8_t* __restrict__ codes,
    float* __restrict__ scales, int64_t ld_codes, typename Elems<DT>::S* __restrict__ sum,
    float* __restrict__ rstd_out, int64_t T, int C, float eps) {
  constexpr int BLOCK = ln_any_block<N>();
  __shared__ float red[BLOCK / kWave];
  __shared__ uint32_t redm[BLOCK / kWave];
  const int lane = static_cast<int>(threadIdx.x);
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    auto load = [&](int c, float (&f)[N]) {
      ln_any_load<DT>(x + t * C + c, f);
      if (r) {
        float g[N];
        ln_any_load<DT>(r + t * C + c, g);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = Elems<DT>::rounded(f[e] + g[e]);
      }
    };
    float s = 0.f, f[N], w[N], rstd = 1.f;
    uint32_t m = 0u;
    for (int i = lane; N * i < C; i += BLOCK) {
      const LnPlace p = ln_any_place<N>(i, C);
      load(p.c, f);
      if constexpr (OUT == kRmsCodes) ln_any_param<DT>(wp, w_f32, p.c, 1.f, w);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = e >= p.skip ? f[e] : 0.f;
        s = __builtin_fmaf(d, d, s);
        const uint32_t bits = __float_as_uint(OUT == kRmsCodes ? f[e] * w[e] : f[e]) & 0x7fffffffu;
        m = bits > m ? bits : m;
      }
    }
    if constexpr (OUT != kRmsRows) rstd = rsqrtf(ln_any_sum<N>(s, red) / static_cast<float>(C) + eps);
    RowScale rs;
    if constexpr (OUT != kRmsY) {
      m = group_max<kWave>(m);
      __syncthreads();  // redm is free again
      if ((lane & (kWave - 1)) == 0) redm[lane >> 6] = m;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < BLOCK / kWave; ++i) m = redm[i] > m ? redm[i] : m;
      rs = row_scale(m, rstd);
    }
    for (int i = lane; N * i < C; i += BLOCK) {
      const LnPlace p = ln_any_place<N>(i, C);
      load(p.c, f);
      if (r) ln_any_store<DT>(sum + t * C + p.c, f);
      if constexpr (OUT != kRmsRows) {
        ln_any_param<DT>(wp, w_f32, p.c, 1.f, w);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = f[e] * rstd * w[e];
      }
      if constexpr (OUT == kRmsY) {
        ln_any_store<DT>(y + t * C + p.c, f);
      } else if constexpr (N == 8) {
        st_codes<false>(codes + t * ld_codes + p.c, row_codes8(f, rs));
      } else {
        codes[t * ld_codes + p.c] = static_cast<int8_t>(row_code(f[0], rs.to_code) & rs.keep);
      }
    }
    if (lane == 0) {
      if constexpr (OUT == kRmsY) {
        if (rstd_out) rstd_out[t] = rstd;
      } else {
        scales[t] = rs.scale;
      }
    }
  }
}

template <int DT, int N>
__global__ __launch_bounds__(ln_any_block<N>()) void rms_bwd_any(
    const typename Elems<DT>::S* __restrict__ gy, const typename Elems<DT>::S* __restrict__ x,
    const float* __restrict__ rstd_in, const void* __restrict__ wp, bool w_f32,
    const typename Elems<DT>::S* __restrict__ gi, typename Elems<DT>::S* __restrict__ gx, int64_t T, int C) {
  constexpr int BLOCK = ln_any_block<N>();
  __shared__ float red[BLOCK / kWave];
  const int lane = static_cast<int>(threadIdx.x);
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    const float rstd = rstd_in[t];
    // g = gy w and h of the lane's columns from p on.
    float g[N], h[N], w[N];
    auto load = [&](const LnPlace& p) {
      ln_any_load<DT>(gy + t * C + p.c, g);
      ln_any_load<DT>(x + t * C + p.c, h);
      ln_any_param<DT>(wp, w_f32, p.c, 1.f, w);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        g[e] *= w[e];
        h[e] *= rstd;
      }
    };
    float s = 0.f;
    for (int i = lane; N * i < C; i += BLOCK) {
      const LnPlace p = ln_any_place<N>(i, C);
      load(p);
#pragma unroll
      for (int e = 0; e < N; ++e) s = __builtin_fmaf(e >= p.skip ? g[e] : 0.f, h[e], s);
    }
    const float c2 = ln_any_sum<N>(s, red) / static_cast<float>(C) * rstd;
    for (int i = lane; N * i < C; i += BLOCK) {
      const LnPlace p = ln_any_place<N>(i, C);
      load(p);
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = __builtin_fmaf(g[e], rstd, -h[e] * c2);
      if (gi) {
        ln_any_load<DT>(gi + t * C + p.c, h);
#pragma unroll
        for (int e = 0; e < N; ++e) g[e] += h[e];
      }
      ln_any_store<DT>(gx + t * C + p.c, g);
    }
  }
}

// Their grad_w: a workgroup takes 256 N columns and rows blockIdx.y, blockIdx.y +
// gridDim.y, ..., into `partial` as rms_bwd_kernel's workgroup blockIdx.y.
template <int DT, int N>
__global__ __launch_bounds__(kLnColumnsBlock) void rms_columns_any(const typename Elems<DT>::S* __restrict__ gy,
                                                                   const typename Elems<DT>::S* __restrict__ x,
                                                                   const float* __restrict__ rstd_in,
                                                                   float* __restrict__ partial, int64_t T, int C) {
  const int i = static_cast<int>(blockIdx.x) * kLnColumnsBlock + static_cast<int>(threadIdx.x);
  if (N * i >= C) return;
  const LnPlace p = ln_any_place<N>(i, C);
  float dw[N];
#pragma unroll
  for (int e = 0; e < N; ++e) dw[e] = 0.f;
  for (int64_t t = blockIdx.y; t < T; t += gridDim.y) {
    float q[N], h[N];
    ln_any_load<DT>(gy + t * C + p.c, q);
    ln_any_load<DT>(x + t * C + p.c, h);
    const float rstd = rstd_in[t];
#pragma unroll
    for (int e = 0; e < N; ++e) dw[e] = __builtin_fmaf(q[e], h[e] * rstd, dw[e]);
  }
  float* dst = partial + static_cast<int64_t>(blockIdx.y) * ((C + 7) / 8 * 8) + p.c;
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e >= p.skip) dst[e] = dw[e];
}

// grad_w from the workgroups' sums, as ln_reduce_kernel.
template <int DT>
__global__ __launch_bounds__(kLnReduceBlock) void rms_reduce_kernel(const float* __restrict__ partial, int64_t parts,
                                                                    int64_t cols, int C, bool f32,
                                                                    void* __restrict__ gw) {
  constexpr int kVecs = 16, kShares = kLnReduceBlock / kVecs;
  __shared__ f32x4 acc[kShares][kVecs];
  const int v = static_cast<int>(threadIdx.x) % kVecs, share = static_cast<int>(threadIdx.x) / kVecs;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * kVecs + v) * 4;  // of cols, a multiple of 8
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (i < cols) {
    const float* src = partial + i;
#pragma unroll 8
    for (int64_t p = share; p < parts; p += kShares) s += *reinterpret_cast<const f32x4*>(src + p * cols);
  }
  acc[share][v] = s;
  __syncthreads();
  if (share < 8) {
#pragma unroll
    for (int k = 8; k < kShares; k += 8) s += acc[share + k][v];
  }
  __syncthreads();
  if (share < 8) acc[share][v] = s;
  __syncthreads();
  if (share != 0 || i >= cols) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += acc[k][v];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (i + e < C) {
      if (f32)
        static_cast<float*>(gw)[i + e] = s[e];
      else
        Elems<DT>::store(static_cast<typename Elems<DT>::S*>(gw) + i + e, s[e]);
    }
  }
}

}  // namespace

template <int DT>
int rms_fwd_run(const RmsFwdArgs& a, hipStream_t s) {
  using S = typename Elems<DT>::S;
  const auto* x = static_cast<const S*>(a.x);
  const auto* r = static_cast<const S*>(a.r);
  auto* y = static_cast<S*>(a.y);
  auto* sum = static_cast<S*>(a.sum);
  // Packed rows carry no nontemporal hint: their codes are multiplied next, and the row may be that
  // product's residual (pack and product with the hint / without, us: T = 65536, C = 1024 with the norm and
  // the residual 136 / 120, T = 8192, C = 2048 47 / 44).
  const bool nt = y && ln_hint<DT>(a.T, a.C) && a.C % 8 == 0 && aligned16(x) && aligned16(r) && aligned16(y) &&
                  aligned16(sum);
  const bool held = with_ln_walk<(DT == FMHC_DTYPE_F32 ? 3 : 5)>(a.T, a.C, [&](auto walk) {
    constexpr int LPT = decltype(walk)::LPT, R = decltype(walk)::R, BLOCK = ln_fwd_block<LPT>();
    auto launch = [&](auto ntc, auto add, auto out) {
      auto* kernel = &rms_fwd_kernel<DT, LPT, R, decltype(ntc)::value, decltype(add)::value, decltype(out)::value>;
      // Eight workgroups per CU, and from there one row per slot where there is a residual, two otherwise
      // (eight per CU / two rows / one, us, T = 65536, C = 2048: with a residual 183 / 176 / 172, without 95 /
      // 86 / 88, packed 75 / 73 / 78 and with a residual 177 / 171 / 164; T = 262144, C = 1024 423 / 365 / 354
      // and 200 / 172 / 171; T = 8192, C = 8192 100 / 98 / 94 and 49 / 48 / 48).  A launch has fewer than 2^32
      // threads; the workgroups walk the rest of the rows.
      const int64_t want = (a.T + BLOCK / LPT - 1) / (BLOCK / LPT), fit = ((int64_t{1} << 32) - 1) / BLOCK;
      const int64_t some = r ? want : want / 2, many = some > 256 * 8 ? some : 256 * 8, most = many < fit ? many : fit;
      kernel<<<dim3(static_cast<unsigned>(want < most ? want : most)), BLOCK, 0, s>>>(
          x, r, a.w, a.w_f32, y, a.codes, a.scales, a.ld_codes, sum, a.rstd, a.T, a.C, a.eps);
    };
    using std::integral_constant;
    constexpr std::true_type yes;
    constexpr std::false_type no;
    constexpr integral_constant<int, kRmsY> as_y;
    constexpr integral_constant<int, kRmsCodes> as_codes;
    if (!a.norm) launch(no, no, integral_constant<int, kRmsRows>{});
    else if (!y) r ? launch(no, yes, as_codes) : launch(no, no, as_codes);
    else if (nt) r ? launch(yes, yes, as_y) : launch(yes, no, as_y);
    else r ? launch(no, yes, as_y) : launch(no, no, as_y);
  });
  if (!held) {
    const int64_t most = 16384;
    auto any = [&](auto n, auto out) {
      constexpr int N = decltype(n)::value;
      rms_fwd_any<DT, N, decltype(out)::value>
          <<<dim3(static_cast<unsigned>(a.T < most ? a.T : most)), ln_any_block<N>(), 0, s>>>(
              x, r, a.w, a.w_f32, y, a.codes, a.scales, a.ld_codes, sum, a.rstd, a.T, a.C, a.eps);
    };
    using std::integral_constant;
    auto pick = [&](auto n) {
      if (!a.norm) any(n, integral_constant<int, kRmsRows>{});
      else if (y) any(n, integral_constant<int, kRmsY>{});
      else any(n, integral_constant<int, kRmsCodes>{});
    };
    a.C < 8 ? pick(integral_constant<int, 1>{}) : pick(integral_constant<int, 8>{});
  }
  return launch_status();
}

template <int DT>
int rms_bwd_run(const RmsBwdArgs& a, hipStream_t s) {
  using S = typename Elems<DT>::S;
  const auto* gy = static_cast<const S*>(a.gy);
  const auto* x = static_cast<const S*>(a.x);
  const auto* gi = static_cast<const S*>(a.gi);
  auto* gx = static_cast<S*>(a.gx);
  int64_t parts = 0;
  static_assert(ln_most_rounds<3, 512>() * 512 * 8 == kRmsHeld);  // with_ln_walk's widest rows
  const bool nt = ln_hint<DT>(a.T, a.C) && a.C % 8 == 0 && aligned16(gy) && aligned16(x) && aligned16(gx) && aligned16(gi);
  const bool held = with_ln_walk<3>(a.T, a.C, [&](auto walk) {
    constexpr int LPT = decltype(walk)::LPT, R = decltype(walk)::R, SLOTS = kLnBwdBlock / LPT;
    const int64_t want = (a.T + SLOTS - 1) / SLOTS;
    // Two workgroups per CU where a lane has one group and no second gradient, otherwise one (one / two,
    // us: T = 65536, C = 512 36.5 / 33.2, with a second gradient 43.5 / 45.9; C = 2048 128.6 / 132.4 and
    // 167.5 / 167.5; T = 16384, C = 1024 18.8 / 18.5 and 23.4 / 25.1; T = 262144, C = 1024 280 / 295).
    const int64_t most = R == 1 && !gi ? kRmsParts : kRmsParts / 2, room = rms_parts(a.T, a.C);
    parts = want < most ? want : most;
    parts = parts < room ? parts : room;
    const unsigned columns = a.gw && !a.partial ? blocks_for(a.C, kRmsColumns) : 0;
    auto launch = [&](auto ntc, auto add) {
      rms_bwd_kernel<DT, LPT, R, decltype(ntc)::value, decltype(add)::value>
          <<<dim3(static_cast<unsigned>(parts) + columns), kLnBwdBlock, 0, s>>>(
              gy, x, a.rstd, a.w, a.w_f32, gi, gx, a.partial, a.gw, static_cast<int>(columns), a.T, a.C);
    };
    auto pick = [&](auto ntc) { gi ? launch(ntc, std::true_type{}) : launch(ntc, std::false_type{}); };
    nt ? pick(std::true_type{}) : pick(std::false_type{});
  });
  if (!held) {
    auto any = [&](auto n) {
      constexpr int N = decltype(n)::value;
      const int64_t most = 16384;
      rms_bwd_any<DT, N><<<dim3(static_cast<unsigned>(a.T < most ? a.T : most)), ln_any_block<N>(), 0, s>>>(
          gy, x, a.rstd, a.w, a.w_f32, gi, gx, a.T, a.C);
      if (!a.partial) return;
      // Four workgroups per CU: each writes sums of all its columns.
      static_assert(kLnColumnsBlock == 256);
      const unsigned blocks = blocks_for(a.C, kLnColumnsBlock * N);
      parts = rms_parts(a.T, a.C);
      rms_columns_any<DT, N><<<dim3(blocks, static_cast<unsigned>(parts)), kLnColumnsBlock, 0, s>>>(
          gy, x, a.rstd, a.partial, a.T, a.C);
    };
    a.C < 8 ? any(std::integral_constant<int, 1>{}) : any(std::integral_constant<int, 8>{});
  }
  const int st = launch_status();
  if (st != FMHC_OK || !a.partial) return st;
  const int64_t cols = rms_cols(a.C);
  rms_reduce_kernel<DT><<<dim3(blocks_for(cols, 64)), kLnReduceBlock, 0, s>>>(a.partial, parts, cols, a.C, a.w_f32, a.gw);
  return launch_status();
}

}  // namespace fmhc
