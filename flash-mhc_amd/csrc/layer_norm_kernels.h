// The layer norm's kernels, for the translation unit of one storage type.
//
// A row is held by LPT lanes, R groups of 8 columns each, from its loads to its
// stores; a lane keeps the same columns for every row of its workgroup, so the
// weight and bias and (backward) the sums of grad_w and grad_b stay in registers.
// The next row's loads are issued before the current row is computed.
// Bound by HBM (some 10 VALU operations per element): T = 65536, C = 2048 in bf16 the
// forward takes 92 us (5.8 TB/s; packed 117, 5.8), the backward 131 + 4.6 for the
// parameters' sums (6.1; from codes 106, 6.4).
// The lane at a row's end with fewer than 8 columns left takes the row's last 8
// instead: every load is one vector inside the row, sums leave out the columns
// that the lane before holds too, and stores write those once more with the
// same values.
#pragma once

#include "layer_norm.h"

namespace fmhc {

namespace {

// 8 elements as loaded.
template <int DT>
struct LnRaw {
  u32x4 a;
};
template <>
struct LnRaw<FMHC_DTYPE_F32> {
  u32x4 a, b;
};

template <int DT, bool NT>
__device__ __forceinline__ LnRaw<DT> ln_load(const typename Elems<DT>::S* p) {
  LnRaw<DT> r;
  r.a = NT ? ld16_stream(p) : ld16(p);
  if constexpr (DT == FMHC_DTYPE_F32) r.b = NT ? ld16_stream(p + 4) : ld16(p + 4);
  return r;
}
template <int DT>
__device__ __forceinline__ void ln_unpack(const LnRaw<DT>& r, float (&f)[8]) {
  if constexpr (DT == FMHC_DTYPE_BF16) {
    unpack8(r.a, f);
  } else if constexpr (DT == FMHC_DTYPE_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = Elems<DT>::widen(r.a[i] & 0xffffu);
      f[2 * i + 1] = Elems<DT>::widen(r.a[i] >> 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = __uint_as_float(r.a[i]);
      f[4 + i] = __uint_as_float(r.b[i]);
    }
  }
}

// A value that the compiler takes as new.
template <int DT>
__device__ __forceinline__ void ln_opaque(LnRaw<DT>& r) {
  asm volatile("" : "+v"(r.a.x), "+v"(r.a.y), "+v"(r.a.z), "+v"(r.a.w));
  if constexpr (DT == FMHC_DTYPE_F32) asm volatile("" : "+v"(r.b.x), "+v"(r.b.y), "+v"(r.b.z), "+v"(r.b.w));
}

// x in the backward: as it is, or codes with their group's scale.
template <int DT, bool KEPT>
struct LnX {
  using Elem = typename Elems<DT>::S;
  LnRaw<DT> r;
};
template <int DT>
struct LnX<DT, true> {
  using Elem = int8_t;
  u32x2 q;
  uint32_t e0, e1;  // the first and the last column's (a lane's last group only)
};

// The values of 8 codes from column c on, in one group for round k < R - 1 and
// in rows of whole groups of 8 (NT).
template <int R, bool NT>
__device__ __forceinline__ void ln_decode(u32x2 q, uint32_t e0, uint32_t e1, int k, int c, float (&f)[8]) {
  if (NT || k < R - 1)
    decode8(q, pack_unit(e0), f);
  else
    decode8(q, pack_unit(e0), pack_unit(e1), kPackGroup - (c & (kPackGroup - 1)), f);
}

// Where lane group g of a row of C >= 8 columns is: 8 columns from `c` on, of
// which the first `skip` belong to the group before (8: the group is past the
// row's end).
struct LnPlace {
  int c, skip;
};
__device__ __forceinline__ LnPlace ln_place(int g, int C) {
  const int c0 = 8 * g, c = c0 < C - 8 ? c0 : C - 8;
  return LnPlace{c, c0 - c < 8 ? c0 - c : 8};
}

template <int DT>
__device__ __forceinline__ void ln_param8(const void* p, bool f32, int c, float none, float (&f)[8]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = none;
  } else if (f32) {
    Elems<FMHC_DTYPE_F32>::load8<false>(static_cast<const float*>(p) + c, f);
  } else {
    Elems<DT>::template load8<false>(static_cast<const typename Elems<DT>::S*>(p) + c, f);
  }
}

// Sums over a row's LPT lanes of a workgroup of BLOCK threads, in every lane.
// With several waves per row their sums go through `red` in wave order; the two
// halves of `red` take turns, so one barrier is enough: a wave writes a half
// again only behind the other half's barrier, which every reader has passed.
template <int LPT, int BLOCK, int N>
struct LnSums {
  static constexpr int WPR = LPT > kWave ? LPT / kWave : 1;
  float (*red)[BLOCK / kWave][N];  // [2]
  int half = 0;
  __device__ __forceinline__ void operator()(float (&v)[N]) {
    if constexpr (WPR == 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = group_sum<LPT>(v[i]);
    } else {
      const int wave = static_cast<int>(threadIdx.x) >> 6;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
      if ((threadIdx.x & (kWave - 1)) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) red[half][wave][i] = v[i];
      }
      __syncthreads();
      const int first = wave & ~(WPR - 1);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = red[half][first][i];
#pragma unroll
        for (int w = 1; w < WPR; ++w) v[i] += red[half][first + w][i];
      }
      half ^= 1;
    }
  }
};

constexpr int kLnFwdBlock = 256;
constexpr int kLnBwdBlock = 512;

// Threads of a forward workgroup: a row's lanes fit.
template <int LPT>
constexpr int ln_fwd_block() {
  return LPT > kLnFwdBlock ? LPT : kLnFwdBlock;
}

template <int DT, int LPT, int R, bool NT, bool KEEP>
__global__ __launch_bounds__(ln_fwd_block<LPT>()) void ln_fwd_kernel(
    const typename Elems<DT>::S* __restrict__ x, const LnParams P, typename Elems<DT>::S* __restrict__ y,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, int8_t* __restrict__ codes,
    uint8_t* __restrict__ scales, int64_t T, int C, float eps) {
  constexpr int BLOCK = ln_fwd_block<LPT>(), SLOTS = BLOCK / LPT;
  __shared__ float red[2][BLOCK / kWave][1];
  LnSums<LPT, BLOCK, 1> row_sum{red};
  const int sub = static_cast<int>(threadIdx.x) % LPT, slot = static_cast<int>(threadIdx.x) / LPT;
  const int G = pack_groups(C);
  const float n_inv = 1.f / static_cast<float>(C);

  LnPlace at[R];
  float w[R][8], b[R][8];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    at[k] = ln_place(sub + k * LPT, C);
    ln_param8<DT>(P.w, P.f32, at[k].c, 1.f, w[k]);
    ln_param8<DT>(P.b, P.f32, at[k].c, 0.f, b[k]);
  }
  // Only a lane's last group can be short or past the row's end.
  auto inside = [&](int k, int e) { return k < R - 1 || e >= at[k].skip; };

  // Every thread walks as many rows (the barriers of LnSums), those past the
  // last one on the last one's data, without storing.
  const int64_t step = static_cast<int64_t>(gridDim.x) * SLOTS;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * SLOTS;
  LnRaw<DT> raw[R];
  auto load = [&](int64_t t) {
    const auto* row = x + (t < T ? t : T - 1) * C;
#pragma unroll
    for (int k = 0; k < R; ++k) raw[k] = ln_load<DT, NT>(row + at[k].c);
  };
  load(first + slot);
  for (int64_t t0 = first; t0 < T; t0 += step) {
    const int64_t t = t0 + slot;
    float v[R][8];
#pragma unroll
    for (int k = 0; k < R; ++k) ln_unpack<DT>(raw[k], v[k]);
    if (t0 + step < T) load(t + step);
    __builtin_amdgcn_sched_barrier(0);

    uint32_t E[R];
    if constexpr (KEEP) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        uint32_t m = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t bits = inside(k, e) ? __float_as_uint(v[k][e]) & 0x7fffffffu : 0u;
          m = bits > m ? bits : m;
        }
        E[k] = pack_scale(quad_max(m));
      }
    }
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] += inside(k, e) ? v[k][e] : 0.f;
    row_sum(s);
    // Divided, not multiplied with 1 / C: the mean of equal values is that value.
    const float mean = s[0] / static_cast<float>(C);
    float s2[1] = {0.f};
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = inside(k, e) ? v[k][e] - mean : 0.f;
        s2[0] = __builtin_fmaf(d, d, s2[0]);
      }
    row_sum(s2);
    const float rstd = rsqrtf(s2[0] * n_inv + eps);
    if (t < T) {
      auto* out = y + t * C;
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (k == R - 1 && at[k].skip == 8) continue;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = __builtin_fmaf((v[k][e] - mean) * rstd, w[k][e], b[k][e]);
        Elems<DT>::template store8<NT>(out + at[k].c, o);
        if constexpr (KEEP) {
          const u32x2 q = encode8(v[k], E[k]);
          int8_t* dst = codes + t * C + at[k].c;
          if (k < R - 1 || at[k].skip == 0) {
            st_codes<NT>(dst, q);
          } else {
            st_last_codes(dst + at[k].skip, q, 8 - at[k].skip);
          }
          const int g = sub + k * LPT;
          if ((g & 3) == 0) scales[t * G + (g >> 2)] = static_cast<uint8_t>(E[k]);
        }
      }
      if (sub == 0) {
        if (mean_out) mean_out[t] = mean;
        if (rstd_out) rstd_out[t] = rstd;
      }
    }
  }
}

// The residual around a norm gives x a second gradient.  With GI it is added here,
// to the rounded one, as adding the two tensors would: that pass reads both and
// writes their sum, here one is read (MHCLiteBlock with pre_norm).
template <int DT, int N>
__device__ __forceinline__ void ln_add_grad(const float (&gi)[N], float (&o)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = gi[e] + Elems<DT>::rounded(o[e]);
}

// partial (may be null): this workgroup's sums, [2][ln_cols(C)]: grad_w, grad_b.
template <int DT, int LPT, int R, bool NT, bool KEPT, bool GI>
__global__ __launch_bounds__(kLnBwdBlock) void ln_bwd_kernel(
    const typename Elems<DT>::S* __restrict__ gy, const typename LnX<DT, KEPT>::Elem* __restrict__ x,
    const uint8_t* __restrict__ scales, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
    const LnParams P, const typename Elems<DT>::S* __restrict__ gi, typename Elems<DT>::S* __restrict__ gx,
    float* __restrict__ partial, int64_t T, int C) {
  constexpr int BLOCK = kLnBwdBlock, SLOTS = BLOCK / LPT;
  __shared__ float red[2][BLOCK / kWave][2];
  LnSums<LPT, BLOCK, 2> row_sums{red};
  const int sub = static_cast<int>(threadIdx.x) % LPT, slot = static_cast<int>(threadIdx.x) / LPT;
  const int G = pack_groups(C);
  const float n_inv = 1.f / static_cast<float>(C);

  LnPlace at[R];
  float w[R][8], dw[R][8], db[R][8];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    at[k] = ln_place(sub + k * LPT, C);
    ln_param8<DT>(P.w, P.f32, at[k].c, 1.f, w[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[k][e] = db[k][e] = 0.f;
  }

  const int64_t step = static_cast<int64_t>(gridDim.x) * SLOTS;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * SLOTS;
  LnRaw<DT> rg[R];
  LnX<DT, KEPT> rx[R];
  LnRaw<DT> ri[GI ? R : 1];
  float mean_n, rstd_n;
  auto load = [&](int64_t tt) {
    const int64_t t = tt < T ? tt : T - 1;
    const auto* grow = gy + t * C;
    const auto* xrow = x + t * C;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      rg[k] = ln_load<DT, NT>(grow + at[k].c);
      if constexpr (KEPT) {
        rx[k].q = ld_codes<NT>(xrow + at[k].c);
        rx[k].e0 = scales[t * G + (at[k].c >> 5)];
        // Eight columns off a multiple of 8 may end in another group of 32.
        rx[k].e1 = NT || k < R - 1 ? rx[k].e0 : scales[t * G + ((at[k].c + 7) >> 5)];
      } else {
        rx[k].r = ln_load<DT, NT>(xrow + at[k].c);
      }
      if constexpr (GI) ri[k] = ln_load<DT, NT>(gi + t * C + at[k].c);
    }
    mean_n = mean_in[t];
    rstd_n = rstd_in[t];
  };
  load(first + slot);
  for (int64_t t0 = first; t0 < T; t0 += step) {
    const int64_t t = t0 + slot;
    const float mean = mean_n, rstd = rstd_n;
    // Few groups per lane stay in fp32 between the sums and the stores; more
    // stay as loaded and are widened again (16 VGPRs of the 61 per group).
    constexpr bool HOLD = R <= 3;
    LnRaw<DT> cg[R];
    LnX<DT, KEPT> cx[R];
    LnRaw<DT> ci[GI ? R : 1];
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
      if constexpr (KEPT)
        ln_decode<R, NT>(cx[k].q, cx[k].e0, cx[k].e1, k, at[k].c, hk);
      else
        ln_unpack<DT>(cx[k].r, hk);
#pragma unroll
      for (int e = 0; e < 8; ++e) hk[e] = (hk[e] - mean) * rstd;
    };

    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float (&qk)[8] = q[HOLD ? k : 0];
      float (&hk)[8] = h[HOLD ? k : 0];
      widen(k, qk, hk);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float g = k < R - 1 || e >= at[k].skip ? qk[e] * w[k][e] : 0.f;
        s[0] += g;
        s[1] = __builtin_fmaf(g, hk[e], s[1]);
      }
    }
    row_sums(s);
    if constexpr (!HOLD) {
      // The compiler is not to keep the widened values after all.
#pragma unroll
      for (int k = 0; k < R; ++k) {
        ln_opaque(cg[k]);
        if constexpr (KEPT)
          asm volatile("" : "+v"(cx[k].q.x), "+v"(cx[k].q.y));
        else
          ln_opaque(cx[k].r);
      }
    }
    if (t < T) {
      // rstd (g - c1 - h c2)
      const float k1 = s[0] * n_inv * rstd, k2 = s[1] * n_inv * rstd;
      auto* out = gx + t * C;
#pragma unroll
      for (int k = 0; k < R; ++k) {
        float (&qk)[8] = q[HOLD ? k : 0];
        float (&hk)[8] = h[HOLD ? k : 0];
        if constexpr (!HOLD) widen(k, qk, hk);
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          o[e] = __builtin_fmaf(-hk[e], k2, __builtin_fmaf(qk[e] * w[k][e], rstd, -k1));
          dw[k][e] = __builtin_fmaf(qk[e], hk[e], dw[k][e]);
          db[k][e] += qk[e];
        }
        if constexpr (GI) {
          float f[8];
          ln_unpack<DT>(ci[k], f);
          ln_add_grad<DT>(f, o);
        }
        if (k < R - 1 || at[k].skip < 8) Elems<DT>::template store8<NT>(out + at[k].c, o);
      }
    }
  }
  if (!partial) return;
  // The workgroup's rows: the threads that hold the same columns, in slot order.
  constexpr int kPitch = BLOCK + 4;
  __shared__ float acc[16 * kPitch];
  const int64_t cols = (C + 7) / 8 * 8;
  float* dst = partial + static_cast<int64_t>(blockIdx.x) * 2 * cols;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      acc[e * kPitch + threadIdx.x] = dw[k][e];
      acc[(8 + e) * kPitch + threadIdx.x] = db[k][e];
    }
    __syncthreads();
    for (int i = static_cast<int>(threadIdx.x); i < 16 * LPT; i += BLOCK) {
      const int which = i / (8 * LPT), j = i % (8 * LPT), own = j / 8, e = j % 8;
      const float* src = acc + (8 * which + e) * kPitch + own;
      float v = src[0];
#pragma unroll
      for (int sl = 1; sl < SLOTS; ++sl) v += src[sl * LPT];
      const LnPlace p = ln_place(own + k * LPT, C);
      if (e >= p.skip) dst[which * cols + p.c + e] = v;
    }
  }
}

// ---------------------------------------------------------------------------
// Rows of fewer than 8 columns (N = 1 at a time, one wave), and rows that no
// registers hold (N = 8, sixteen waves): one workgroup per row, which is read
// again for every use, from L2.  T = 2000, C = 20000 in bf16: 48 us forward, 91
// backward (one element at a time and four waves: 137 and 138).
template <int N>
constexpr int ln_any_block() {
  return N == 8 ? 1024 : kWave;
}
constexpr int kLnColumnsBlock = 256;

template <int N>
__device__ __forceinline__ float ln_any_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();  // red is free again
  if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int i = 1; i < ln_any_block<N>() / kWave; ++i) s += red[i];
  return s;
}

// The lane's i-th N columns of a row.
template <int N>
__device__ __forceinline__ LnPlace ln_any_place(int i, int C) {
  if constexpr (N == 8)
    return ln_place(i, C);
  else
    return LnPlace{i, 0};
}

template <int DT, int N>
__device__ __forceinline__ void ln_any_load(const typename Elems<DT>::S* p, float (&f)[N]) {
  if constexpr (N == 8)
    Elems<DT>::template load8<false>(p, f);
  else
    f[0] = Elems<DT>::load(p);
}
template <int DT, int N>
__device__ __forceinline__ void ln_any_store(typename Elems<DT>::S* p, const float (&f)[N]) {
  if constexpr (N == 8)
    Elems<DT>::template store8<false>(p, f);
  else
    Elems<DT>::store(p, f[0]);
}

template <int DT, int N>
__device__ __forceinline__ void ln_any_param(const void* p, bool f32, int c, float none, float (&f)[N]) {
  if constexpr (N == 8)
    ln_param8<DT>(p, f32, c, none, f);
  else if (!p)
    f[0] = none;
  else
    f[0] = f32 ? static_cast<const float*>(p)[c] : Elems<DT>::load(static_cast<const typename Elems<DT>::S*>(p) + c);
}

// x[t, c .. c + N) in the backward.
template <int DT, bool KEPT, int N>
__device__ __forceinline__ void ln_any_x(const typename LnX<DT, KEPT>::Elem* x, const uint8_t* scales, int64_t t, int c,
                                         int C, float (&f)[N]) {
  if constexpr (KEPT) {
    const uint8_t* row = scales + t * pack_groups(C);
    if constexpr (N == 8)
      decode8(ld_codes<false>(x + t * C + c), pack_unit(row[c >> 5]), pack_unit(row[(c + 7) >> 5]),
              kPackGroup - (c & (kPackGroup - 1)), f);
    else
      f[0] = static_cast<float>(x[t * C + c]) * pack_unit(row[c >> 5]);
  } else {
    ln_any_load<DT>(x + t * C + c, f);
  }
}

template <int DT, int N>
__global__ __launch_bounds__(ln_any_block<N>()) void ln_fwd_any(const typename Elems<DT>::S* __restrict__ x, const LnParams P,
                                                          typename Elems<DT>::S* __restrict__ y,
                                                          float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                          int8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                          int64_t T, int C, float eps) {
  __shared__ float red[ln_any_block<N>() / kWave];
  const int lane = static_cast<int>(threadIdx.x);
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    const auto* row = x + t * C;
    float s = 0.f, s2 = 0.f, f[N], w[N], b[N];
    for (int i = lane; N * i < C; i += ln_any_block<N>()) {
      const LnPlace p = ln_any_place<N>(i, C);
      ln_any_load<DT>(row + p.c, f);
#pragma unroll
      for (int e = 0; e < N; ++e) s += e >= p.skip ? f[e] : 0.f;
    }
    const float mean = ln_any_sum<N>(s, red) / static_cast<float>(C);
    for (int i = lane; N * i < C; i += ln_any_block<N>()) {
      const LnPlace p = ln_any_place<N>(i, C);
      ln_any_load<DT>(row + p.c, f);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = e >= p.skip ? f[e] - mean : 0.f;
        s2 = __builtin_fmaf(d, d, s2);
      }
    }
    const float rstd = rsqrtf(ln_any_sum<N>(s2, red) / static_cast<float>(C) + eps);
    for (int i = lane; N * i < C; i += ln_any_block<N>()) {
      const LnPlace p = ln_any_place<N>(i, C);
      ln_any_load<DT>(row + p.c, f);
      ln_any_param<DT>(P.w, P.f32, p.c, 1.f, w);
      ln_any_param<DT>(P.b, P.f32, p.c, 0.f, b);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = __builtin_fmaf((f[e] - mean) * rstd, w[e], b[e]);
      ln_any_store<DT>(y + t * C + p.c, f);
    }
    if (codes) {
      // A lane takes 8 columns, a quad of lanes a group of 32.
      for (int g = lane; (g & ~3) < 4 * pack_groups(C); g += ln_any_block<N>()) {
        float v[8];
        if (8 * g + 8 <= C) {
          Elems<DT>::template load8<false>(row + 8 * g, v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = 8 * g + e < C ? Elems<DT>::load(row + 8 * g + e) : 0.f;
        }
        const uint32_t E = pack_scale(quad_max(max_bits8(v)));
        const u32x2 q = encode8(v, E);
        if (8 * g + 8 <= C) {
          st_codes<false>(codes + t * C + 8 * g, q);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (8 * g + e < C) codes[t * C + 8 * g + e] = static_cast<int8_t>(q[e >> 2] >> (8 * (e & 3)));
        }
        if ((g & 3) == 0 && 8 * g < C) scales[t * pack_groups(C) + (g >> 2)] = static_cast<uint8_t>(E);
      }
    }
    if (lane == 0) {
      if (mean_out) mean_out[t] = mean;
      if (rstd_out) rstd_out[t] = rstd;
    }
  }
}

template <int DT, bool KEPT, int N>
__global__ __launch_bounds__(ln_any_block<N>()) void ln_bwd_any(const typename Elems<DT>::S* __restrict__ gy,
                                                          const typename LnX<DT, KEPT>::Elem* __restrict__ x,
                                                          const uint8_t* __restrict__ scales,
                                                          const float* __restrict__ mean_in,
                                                          const float* __restrict__ rstd_in, const LnParams P,
                                                          const typename Elems<DT>::S* __restrict__ gi,
                                                          typename Elems<DT>::S* __restrict__ gx, int64_t T, int C) {
  __shared__ float red[ln_any_block<N>() / kWave];
  const int lane = static_cast<int>(threadIdx.x);
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    const float mean = mean_in[t], rstd = rstd_in[t];
    // g = gy w and h of the lane's columns from p on.
    float g[N], h[N], w[N];
    auto load = [&](const LnPlace& p) {
      ln_any_load<DT>(gy + t * C + p.c, g);
      ln_any_x<DT, KEPT>(x, scales, t, p.c, C, h);
      ln_any_param<DT>(P.w, P.f32, p.c, 1.f, w);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        g[e] *= w[e];
        h[e] = (h[e] - mean) * rstd;
      }
    };
    float s1 = 0.f, s2 = 0.f;
    for (int i = lane; N * i < C; i += ln_any_block<N>()) {
      const LnPlace p = ln_any_place<N>(i, C);
      load(p);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float v = e >= p.skip ? g[e] : 0.f;
        s1 += v;
        s2 = __builtin_fmaf(v, h[e], s2);
      }
    }
    const float c1 = ln_any_sum<N>(s1, red) / static_cast<float>(C), c2 = ln_any_sum<N>(s2, red) / static_cast<float>(C);
    for (int i = lane; N * i < C; i += ln_any_block<N>()) {
      const LnPlace p = ln_any_place<N>(i, C);
      load(p);
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = rstd * (g[e] - c1 - h[e] * c2);
      if (gi) {
        ln_any_load<DT>(gi + t * C + p.c, h);
        ln_add_grad<DT>(h, g);
      }
      ln_any_store<DT>(gx + t * C + p.c, g);
    }
  }
}

// Their grad_w and grad_b: a workgroup takes 256 N columns and rows blockIdx.y,
// blockIdx.y + gridDim.y, ..., into `partial` as ln_bwd_kernel's workgroup
// blockIdx.y.
template <int DT, bool KEPT, int N>
__global__ __launch_bounds__(kLnColumnsBlock) void ln_columns_any(const typename Elems<DT>::S* __restrict__ gy,
                                                              const typename LnX<DT, KEPT>::Elem* __restrict__ x,
                                                              const uint8_t* __restrict__ scales,
                                                              const float* __restrict__ mean_in,
                                                              const float* __restrict__ rstd_in,
                                                              float* __restrict__ partial, int64_t T, int C) {
  const int64_t cols = (C + 7) / 8 * 8;
  const int i = static_cast<int>(blockIdx.x) * kLnColumnsBlock + static_cast<int>(threadIdx.x);
  if (N * i >= C) return;
  const LnPlace p = ln_any_place<N>(i, C);
  float dw[N], db[N];
#pragma unroll
  for (int e = 0; e < N; ++e) dw[e] = db[e] = 0.f;
  for (int64_t t = blockIdx.y; t < T; t += gridDim.y) {
    float q[N], h[N];
    ln_any_load<DT>(gy + t * C + p.c, q);
    ln_any_x<DT, KEPT>(x, scales, t, p.c, C, h);
    const float mean = mean_in[t], rstd = rstd_in[t];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      dw[e] = __builtin_fmaf(q[e], (h[e] - mean) * rstd, dw[e]);
      db[e] += q[e];
    }
  }
  float* dst = partial + static_cast<int64_t>(blockIdx.y) * 2 * cols + p.c;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    if (e >= p.skip) {
      dst[e] = dw[e];
      dst[cols + e] = db[e];
    }
  }
}

// grad_w and grad_b from the workgroups' sums: 16 vectors of four columns per
// workgroup, 64 shares of the parts, added in order.  A chain of load latencies:
// with 16 shares a thread walks up to 32 parts.
constexpr int kLnReduceBlock = 1024;
template <int DT>
__global__ __launch_bounds__(kLnReduceBlock) void ln_reduce_kernel(const float* __restrict__ partial, int64_t parts,
                                                                   int64_t cols, int C, bool f32,
                                                                   void* __restrict__ gw, void* __restrict__ gb) {
  constexpr int kVecs = 16, kShares = kLnReduceBlock / kVecs;
  __shared__ f32x4 acc[kShares][kVecs];
  const int v = static_cast<int>(threadIdx.x) % kVecs, share = static_cast<int>(threadIdx.x) / kVecs;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * kVecs + v) * 4;  // of 2 cols, a multiple of 16
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (i < 2 * cols) {
    const float* src = partial + i;
#pragma unroll 8
    for (int64_t p = share; p < parts; p += kShares) s += *reinterpret_cast<const f32x4*>(src + p * 2 * cols);
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
  if (share != 0 || i >= 2 * cols) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += acc[k][v];
  void* dst = i < cols ? gw : gb;
  if (!dst) return;
  const int64_t c = i < cols ? i : i - cols;
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

// ---------------------------------------------------------------------------
// How rows are laid over lanes.

template <int kLpt, int kR>
struct LnWalk {
  static constexpr int LPT = kLpt, R = kR;
};

// Groups per lane at most with LPT lanes per row, where RMAX fit: five only with
// up to two waves per row, four always with eight (no more lanes to take).
template <int RMAX, int LPT>
constexpr int ln_most_rounds() {
  return LPT == 512 ? 4 : LPT <= 128 || RMAX < 4 ? RMAX : 4;
}

// f(LnWalk) for T rows of C columns, 8 or more, held by registers with at most
// RMAX groups per lane; false where there is no such layout.
//
// Many rows take few lanes each: one wave sums a row without LDS and a barrier.
// Few rows take more, so that every CU has some.  Forward, bf16, fewer lanes / more
// (us): C = 2048 T = 64 3.9 / 3.3, T = 65536 94 / 99; C = 1536 T = 1024 3.9 / 3.9, T =
// 4096 6.3 / 8.0; C = 4096 (128 lanes, 256) T = 4096 16.4 / 14.1, T = 8192 24.8 /
// 24.9, T = 16384 47.8 / 48.6; C = 8192 (256, 512) T = 256 4.7 / 4.3, T = 1024 9.3 /
// 9.6, T = 4096 25.4 / 28.1.  The backward differs by 2% at most.
//
// RMAX: five groups per lane forward in 16-bit types (C = 2560, T = 65536, three
// instead 117 -> 119, packed 155 -> 163), three in fp32 (four: T = 32768, C = 2048 95
// -> 102) and in the backward (five: beyond the registers).  320 lanes for rows of 257
// to 320 groups, none idle: C = 2560, T = 65536 114 -> 126 forward, 167 -> 176 backward.
template <int RMAX, typename F>
bool with_ln_walk(int64_t T, int C, F&& f) {
  if (C < 8) return false;
  const int groups = (C + 7) / 8;
  auto rounds = [&](auto lpt, bool may) {
    constexpr int L = decltype(lpt)::value, most = ln_most_rounds<RMAX, L>();
    static_assert(most >= 3 && most <= 5);
    const int r = (groups + L - 1) / L;
    if (!may || r > most) return false;
    if (r == 1) f(LnWalk<L, 1>{});
    else if (r == 2) f(LnWalk<L, 2>{});
    else if (r == 3) f(LnWalk<L, 3>{});
    else if constexpr (most >= 4) {
      if (r == 4) f(LnWalk<L, 4>{});
      else if constexpr (most >= 5) f(LnWalk<L, 5>{});
    }
    return true;
  };
  using std::integral_constant;
  if (groups <= 8) f(LnWalk<8, 1>{});
  else if (groups <= 16) f(LnWalk<16, 1>{});
  else if (groups <= 32) f(LnWalk<32, 1>{});
  else if (groups <= 64) f(LnWalk<64, 1>{});
  else return rounds(integral_constant<int, 64>{}, groups <= 128 || T >= 1024) ||
              rounds(integral_constant<int, 128>{}, groups <= 256 || T >= 8192) ||
              rounds(integral_constant<int, 256>{}, groups <= 512 || T >= 512) ||
              rounds(integral_constant<int, 512>{}, true);
  return true;
}

// Whether whole aligned rows carry the nontemporal hint.  In fp32, whose loads take
// half a lane's columns each, only rows of more than one group per lane in up to
// 256 MiB (hint / none, us, forward and backward: T = 32768, C = 2048 95 / 98 and 141
// / 151, T = 65536, C = 1024 97 / 100 and 150 / 149; T = 131072, C = 1024 213 / 197
// and 313 / 294, C = 320 74 / 68 and 106 / 103).
template <int DT>
bool ln_hint(int64_t T, int C) {
  return DT != FMHC_DTYPE_F32 || (C > 512 && T * C <= int64_t{1} << 26);
}

}  // namespace

template <int DT>
int ln_fwd_run(const LnFwdArgs& a, hipStream_t s) {
  using S = typename Elems<DT>::S;
  const auto* x = static_cast<const S*>(a.x);
  auto* y = static_cast<S*>(a.y);
  const bool nt = ln_hint<DT>(a.T, a.C) && a.C % 8 == 0 && aligned16(x) && aligned16(y) &&
                  (!a.codes || Pack8Src::aligned(a.codes));
  const bool held = with_ln_walk<(DT == FMHC_DTYPE_F32 ? 3 : 5)>(a.T, a.C, [&](auto walk) {
    constexpr int LPT = decltype(walk)::LPT, R = decltype(walk)::R, BLOCK = ln_fwd_block<LPT>();
    auto launch = [&](auto ntc, auto keep) {
      constexpr bool NT = decltype(ntc)::value, KEEP = decltype(keep)::value;
      auto* kernel = &ln_fwd_kernel<DT, LPT, R, NT, KEEP>;
      const int64_t want = (a.T + BLOCK / LPT - 1) / (BLOCK / LPT);
      // Eight workgroups per CU; with rows of up to one wave more, from four rows per
      // slot on (T = 262144, C = 1024 202 -> 174 us, T = 65536, C = 2048 94 -> 90; at
      // two rows per slot T = 30011, C = 2560 54 -> 69; with wider rows C = 8192 packed
      // 61 -> 64).
      // A launch has fewer than 2^32 threads; the workgroups walk the rest of the rows.
      const int64_t deep = LPT <= kWave ? want / 4 : 0, fit = ((int64_t{1} << 32) - 1) / BLOCK;
      const int64_t many = deep > 256 * 8 ? deep : 256 * 8, most = many < fit ? many : fit;
      kernel<<<dim3(static_cast<unsigned>(want < most ? want : most)), BLOCK, 0, s>>>(x, a.P, y, a.mean, a.rstd, a.codes,
                                                                                    a.scales, a.T, a.C, a.eps);
    };
    auto pick = [&](auto ntc) { a.codes ? launch(ntc, std::true_type{}) : launch(ntc, std::false_type{}); };
    nt ? pick(std::true_type{}) : pick(std::false_type{});
  });
  if (!held) {
    const int64_t most = 16384;
    auto any = [&](auto n) {
      constexpr int N = decltype(n)::value;
      ln_fwd_any<DT, N><<<dim3(static_cast<unsigned>(a.T < most ? a.T : most)), ln_any_block<N>(), 0, s>>>(
          x, a.P, y, a.mean, a.rstd, a.codes, a.scales, a.T, a.C, a.eps);
    };
    a.C < 8 ? any(std::integral_constant<int, 1>{}) : any(std::integral_constant<int, 8>{});
  }
  return launch_status();
}

template <int DT>
int ln_bwd_run(const LnBwdArgs& a, hipStream_t s) {
  using S = typename Elems<DT>::S;
  const auto* gy = static_cast<const S*>(a.gy);
  const auto* gi = static_cast<const S*>(a.gi);
  auto* gx = static_cast<S*>(a.gx);
  const int64_t cols = ln_cols(a.C);
  int64_t parts = 0;
  auto run = [&](auto kept) {
    constexpr bool KEPT = decltype(kept)::value;
    using X = typename LnX<DT, KEPT>::Elem;
    const X* x = nullptr;
    if constexpr (KEPT)
      x = a.codes;
    else
      x = static_cast<const X*>(a.x);
    const bool nt = ln_hint<DT>(a.T, a.C) && a.C % 8 == 0 && aligned16(gy) && aligned16(gx) && aligned16(gi) &&
                    (reinterpret_cast<uintptr_t>(x) & (KEPT ? 7u : 15u)) == 0;
    const bool held = with_ln_walk<3>(a.T, a.C, [&](auto walk) {
      constexpr int LPT = decltype(walk)::LPT, R = decltype(walk)::R, SLOTS = kLnBwdBlock / LPT;
      const int64_t want = (a.T + SLOTS - 1) / SLOTS;
      const int64_t most = R == 1 ? kLnParts : kLnParts / 2;
      parts = want < most ? want : most;
      auto launch = [&](auto ntc, auto add) {
        ln_bwd_kernel<DT, LPT, R, decltype(ntc)::value, KEPT, decltype(add)::value>
            <<<dim3(static_cast<unsigned>(parts)), kLnBwdBlock, 0, s>>>(gy, x, a.scales, a.mean, a.rstd, a.P, gi, gx,
                                                                        a.partial, a.T, a.C);
      };
      auto pick = [&](auto ntc) { gi ? launch(ntc, std::true_type{}) : launch(ntc, std::false_type{}); };
      nt ? pick(std::true_type{}) : pick(std::false_type{});
    });
    if (!held) {
      auto any = [&](auto n) {
        constexpr int N = decltype(n)::value;
        const int64_t most = 16384;
        ln_bwd_any<DT, KEPT, N><<<dim3(static_cast<unsigned>(a.T < most ? a.T : most)), ln_any_block<N>(), 0, s>>>(
            gy, x, a.scales, a.mean, a.rstd, a.P, gi, gx, a.T, a.C);
        if (!a.partial) return;
        // Four workgroups per CU: each writes sums of all its columns.
        const unsigned blocks = blocks_for(a.C, kLnColumnsBlock * N);
        const int64_t share = 1024 / blocks > 1 ? 1024 / blocks : 1, limit = share < kLnParts ? share : kLnParts;
        parts = a.T < limit ? a.T : limit;
        ln_columns_any<DT, KEPT, N><<<dim3(blocks, static_cast<unsigned>(parts)), kLnColumnsBlock, 0, s>>>(
            gy, x, a.scales, a.mean, a.rstd, a.partial, a.T, a.C);
      };
      a.C < 8 ? any(std::integral_constant<int, 1>{}) : any(std::integral_constant<int, 8>{});
    }
  };
  a.x ? run(std::false_type{}) : run(std::true_type{});
  const int st = launch_status();
  if (st != FMHC_OK || !a.partial) return st;
  ln_reduce_kernel<DT><<<dim3(blocks_for(2 * cols, 64)), kLnReduceBlock, 0, s>>>(a.partial, parts, cols, a.C, a.P.f32,
                                                                                 a.gw, a.gb);
  return launch_status();
}

}  // namespace fmhc
