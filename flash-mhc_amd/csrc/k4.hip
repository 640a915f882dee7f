// K4: post-mixing (residual stream mix + post-weighted layer output) and its
// backward.
//
//   forward   out[t,i,c]    = bf16(h_post[t,i] * lo[t,c] + sum_j H[t,i,j] * x[t,j,c])
//   backward  grad_lo[t,c]  = bf16(sum_i h_post[t,i] * go[t,i,c])
//             grad_hp[t,i]  = sum_c go[t,i,c] * lo[t,c]           (fp32)
//             grad_H[t,i,j] = sum_c go[t,i,c] * x[t,j,c]          (fp32)
//             grad_x[t,j,c] = bf16(sum_i H[t,i,j] * go[t,i,c])
//
// Follows src/flash_mhc/kernels.py:384-481 (forward) and :487-665 (fused
// backward) of the reference, written for gfx950: a group of LPT consecutive
// lanes owns one token and streams 16-byte vectors of every row it touches, so
// each input row is read once and each output row written once per launch.
// The backward keeps its 20 per-token partial sums in registers and finishes
// them with an in-wave butterfly (and, when a token spans several waves, an
// LDS sum over them in wave order): no atomics, deterministic.
#include <type_traits>

#include "fmhc_common.h"
#include "pack8.h"

namespace fmhc {

namespace {

template <typename WALK>
__global__ __launch_bounds__(block_of<WALK::LPT>()) void k4_fwd_kernel(const uint16_t* __restrict__ x,
                                                        const uint16_t* __restrict__ lo,
                                                        const float* __restrict__ H,
                                                        const float* __restrict__ h_post,
                                                        uint16_t* __restrict__ out,
                                                        int64_t T, int C) {
  constexpr int LPT = WALK::LPT;
  constexpr bool LOOP = WALK::LOOP, WHOLE = WALK::WHOLE;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t tok = token_of_lane<LPT>(lane);
  if (tok >= T) return;
  const int sub = sub_of_lane<LPT>();
  const int ng = C / 8;

  float h[4][4], p[4];
  {
    const float* Ht = H + tok * 16;
    const float* pt = h_post + tok * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = pt[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[i][j] = Ht[i * 4 + j];
    }
  }
  const uint16_t* xr[4];
  uint16_t* orow[4];
  xr[0] = x + tok * 4 * C;
  orow[0] = out + tok * 4 * C;
#pragma unroll
  for (int j = 1; j < 4; ++j) {
    xr[j] = xr[j - 1] + C;
    orow[j] = orow[j - 1] + C;
  }
  const uint16_t* lrow = lo + tok * C;

  auto mix = [&](auto vec, int g) __attribute__((always_inline)) {
    constexpr int VEC = decltype(vec)::value;
    float l[VEC], xv[4][VEC];
    Lanes<VEC, WHOLE>::load(lrow, g, l);
#pragma unroll
    for (int j = 0; j < 4; ++j) Lanes<VEC, WHOLE>::load(xr[j], g, xv[j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float acc = p[i] * l[e];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc = __builtin_fmaf(h[i][j], xv[j][e], acc);
        o[e] = acc;
      }
      Lanes<VEC, WHOLE>::store(orow[i], g, o);
    }
  };
  if constexpr (!LOOP) {
    if (sub < ng) mix(Vec<8>{}, sub);
  } else {
#pragma unroll 2
    for (int g = sub; g < ng; g += LPT) mix(Vec<8>{}, g);
  }
  row_tail<WHOLE>(C, sub, [&](int c) { mix(Vec<1>{}, c); });
}

// The forward that also leaves x and lo in 8 bits (pack8.h) for the backward:
// out as k4_fwd_kernel gives it, and the codes and scales of the rows it has in
// registers anyway, which a pass of its own would read again (T = 65536, C = 1024
// 257 us, 6.1 TB/s; the forward alone 184, a pass over x alone 132).  A quad of lanes
// holds a group of 32 columns.  The lane at a row's end with fewer than 8
// columns left takes the row's last 8: it leaves those of the lane before out of
// its group's maximum, and stores them once more with the same values.  SHORT:
// rows of fewer than 8 columns, one element at a time.
// PACKX: x too, not lo alone (a block's pre-map has packed it already).
// RES: lo is round(res + lo), the residual around a block's norm and layer, summed
// here (T = 65536, C = 1024 257 -> 280 us; PyTorch's addition by itself 68).
template <typename WALK, bool SHORT, bool PACKX, bool RES>
__global__ __launch_bounds__(block_of<WALK::LPT>()) void k4_fwd_pack8_kernel(
    const uint16_t* __restrict__ x, const uint16_t* __restrict__ lo, const float* __restrict__ H,
    const float* __restrict__ h_post, uint16_t* __restrict__ out, int8_t* __restrict__ xq, uint8_t* __restrict__ xs,
    int8_t* __restrict__ lq, uint8_t* __restrict__ ls, int64_t T, int C, const uint16_t* __restrict__ res) {
  constexpr int LPT = WALK::LPT;
  constexpr bool LOOP = WALK::LOOP, WHOLE = WALK::WHOLE;
  static_assert(LPT % 4 == 0, "a group's quad of lanes");
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t tok = token_of_lane<LPT>(lane);
  if (tok >= T) return;
  const int sub = sub_of_lane<LPT>();
  const int G = pack_groups(C);

  float h[4][4], p[4];
  {
    const float* Ht = H + tok * 16;
    const float* pt = h_post + tok * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = pt[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[i][j] = Ht[i * 4 + j];
    }
  }
  const uint16_t* x0 = x + tok * 4 * C;
  const uint16_t* lrow = lo + tok * C;
  uint16_t* o0 = out + tok * 4 * C;
  int8_t* q0 = PACKX ? xq + tok * 4 * C : nullptr;
  uint8_t* s0 = PACKX ? xs + tok * 4 * G : nullptr;

  // Lane group g: columns 8 g .. 8 g + 7, of which n are in the row.
  auto round = [&](int g) __attribute__((always_inline)) {
    const int n = C - 8 * g;
    const int c = SHORT || n >= 8 ? 8 * g : C - 8;  // the eight columns it holds
    const int skip = 8 * g - c;                     // (8 or more: past the row's end)
    float v[5][8];                                  // lo, then the streams
    auto fetch = [&](const uint16_t* row, float (&f)[8]) __attribute__((always_inline)) {
      if constexpr (SHORT) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = e < n ? bf16_to_f32(row[c + e]) : 0.f;
      } else {
        Lanes<8, WHOLE>::load(row + c, 0, f);
      }
    };
    float rv[RES ? 8 : 1];
    fetch(lrow, v[0]);
    if constexpr (RES) fetch(res + tok * C, rv);
#pragma unroll
    for (int j = 0; j < 4; ++j) fetch(x0 + j * int64_t{C}, v[1 + j]);
    if constexpr (RES) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[0][e] = bf16_to_f32(f32_to_bf16(rv[e] + v[0][e]));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float acc = p[i] * v[0][e];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc = __builtin_fmaf(h[i][j], v[1 + j][e], acc);
        o[e] = acc;
      }
      uint16_t* orow = o0 + i * int64_t{C};
      if constexpr (SHORT) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) orow[c + e] = f32_to_bf16(o[e]);
      } else if (n > 0) {
        Lanes<8, WHOLE>::store(orow + c, 0, o);
      }
    }
#pragma unroll
    for (int k = 0; k < (PACKX ? 5 : 1); ++k) {
      uint32_t m = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // SHORT: zeros past the end; WHOLE: a lane's columns are its own, or none are in the row.
        const uint32_t b = __float_as_uint(v[k][e]) & 0x7fffffffu;
        const bool own = SHORT || (WHOLE ? n > 0 : e >= skip);
        m = own && b > m ? b : m;
      }
      const uint32_t E = pack_scale(quad_max(m));  // the whole quad is here
      const u32x2 q = encode8(v[k], E);
      int8_t* qrow = k == 0 ? lq + tok * C : q0 + (k - 1) * int64_t{C};
      uint8_t* srow = k == 0 ? ls + tok * G : s0 + (k - 1) * int64_t{G};
      if constexpr (SHORT) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) qrow[c + e] = static_cast<int8_t>(q[e >> 2] >> (8 * (e & 3)));
      } else if (WHOLE ? n > 0 : n >= 8) {
        st_codes<WHOLE>(qrow + c, q);
      } else if (!WHOLE && n > 0) {
        st_last_codes(qrow + 8 * g, q, n);
      }
      if ((g & 3) == 0 && n > 0) srow[g >> 2] = static_cast<uint8_t>(E);
    }
  };
  // Quads enter whole: a quad's first lane holds a group's first columns.
  if constexpr (!LOOP) {
    if ((sub & ~3) < 4 * G) round(sub);
  } else {
    for (int g = sub; (g & ~3) < 4 * G; g += LPT) round(g);
  }
}

// SRC: where x and lo are read from (bf16 rows, or their 8-bit copies with
// scales xs and los; pack8.h).  The arithmetic and the order of the sums are
// the same.  T = 65536, C = 1024 295 us from bf16, 243 from 8 bits (6.4 TB/s).
template <typename WALK, bool EARLY, typename SRC>
__global__ __launch_bounds__(block_of<WALK::LPT>()) void k4_bwd_kernel(const typename SRC::Elem* __restrict__ x,
                                                        const typename SRC::Elem* __restrict__ lo,
                                                        const float* __restrict__ H,
                                                        const float* __restrict__ h_post,
                                                        const uint16_t* __restrict__ go,
                                                        uint16_t* __restrict__ grad_x,
                                                        uint16_t* __restrict__ grad_lo,
                                                        float* __restrict__ grad_H,
                                                        float* __restrict__ grad_hp,
                                                        int64_t T, int C, const uint8_t* __restrict__ xs,
                                                        const uint8_t* __restrict__ los) {
  constexpr int LPT = WALK::LPT;
  constexpr bool LOOP = WALK::LOOP, WHOLE = WALK::WHOLE;
  constexpr int WPT = LPT > kWave ? LPT / kWave : 1;  // waves per token
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t tok = token_of_lane<LPT>(lane);
  // With several waves per token every wave reaches the barrier below.
  if constexpr (WPT == 1) {
    if (tok >= T) return;
  }
  const bool live = tok < T;
  const int sub = sub_of_lane<LPT>();
  const int ng = C / 8;

  float shp[4] = {0.f, 0.f, 0.f, 0.f};
  float sH[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sH[i][j] = 0.f;

  if (live) {
  float h[4][4], p[4];
  {
    const float* Ht = H + tok * 16;
    const float* pt = h_post + tok * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = pt[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[i][j] = Ht[i * 4 + j];
    }
  }
  using Row = typename SRC::template Row<WHOLE>;
  Row xr[4];
  const uint16_t* gr[4];
  uint16_t* gxr[4];
  xr[0] = Row::at(x, xs, tok * 4, C);
  gr[0] = go + tok * 4 * C;
  gxr[0] = grad_x + tok * 4 * C;
#pragma unroll
  for (int j = 1; j < 4; ++j) {
    xr[j] = xr[j - 1].next(C);
    gr[j] = gr[j - 1] + C;
    gxr[j] = gxr[j - 1] + C;
  }
  const Row lrow = Row::at(lo, los, tok, C);
  uint16_t* glrow = grad_lo + tok * C;

  auto round = [&](auto vec, int g) __attribute__((always_inline)) {
    constexpr int VEC = decltype(vec)::value;
    float q[4][VEC], l[VEC];
#pragma unroll
    for (int i = 0; i < 4; ++i) Lanes<VEC, WHOLE>::load(gr[i], g, q[i]);
    lrow.load(g, l);

    // EARLY: the iteration's x rows load with grad_out and lo, before its
    // first store (the compiler keeps a load behind an earlier store).
    float xe[EARLY ? 4 : 1][VEC];
    if constexpr (EARLY) {
#pragma unroll
      for (int j = 0; j < 4; ++j) xr[j].load(g, xe[j]);
    }
    // grad_lo and the grad_h_post partial sums.
    {
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float acc = p[0] * q[0][e];
        acc = __builtin_fmaf(p[1], q[1][e], acc);
        acc = __builtin_fmaf(p[2], q[2][e], acc);
        o[e] = __builtin_fmaf(p[3], q[3][e], acc);
      }
      Lanes<VEC, WHOLE>::store(glrow, g, o);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) shp[i] = __builtin_fmaf(q[i][e], l[e], shp[i]);
    }

    // One x stream at a time: grad_H partial sums and grad_x.
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float xl[VEC], o[VEC];
      const float* xv = xl;
      if constexpr (EARLY)
        xv = xe[j];
      else
        xr[j].load(g, xl);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sH[i][j] = __builtin_fmaf(q[i][e], xv[e], sH[i][j]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float acc = h[0][j] * q[0][e];
        acc = __builtin_fmaf(h[1][j], q[1][e], acc);
        acc = __builtin_fmaf(h[2][j], q[2][e], acc);
        o[e] = __builtin_fmaf(h[3][j], q[3][e], acc);
      }
      Lanes<VEC, WHOLE>::store(gxr[j], g, o);
    }
  };
  if constexpr (!LOOP) {
    if (sub < ng) round(Vec<8>{}, sub);
  } else {
#pragma unroll 2
    for (int g = sub; g < ng; g += LPT) round(Vec<8>{}, g);
  }
  row_tail<WHOLE>(C, sub, [&](int c) { round(Vec<1>{}, c); });
  }

  constexpr int GS = LPT < kWave ? LPT : kWave;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    shp[i] = group_sum<GS>(shp[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) sH[i][j] = group_sum<GS>(sH[i][j]);
  }
  if constexpr (WPT > 1) {
    // The token's waves add their 20 sums in wave order (deterministic).
    __shared__ float red[block_of<LPT>() / kWave][20];
    const int wave = static_cast<int>(threadIdx.x) >> 6;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        red[wave][16 + i] = shp[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) red[wave][i * 4 + j] = sH[i][j];
      }
    }
    __syncthreads();
    if (live && sub == 0) {
      float t[20];
#pragma unroll
      for (int k = 0; k < 20; ++k) t[k] = 0.f;
#pragma unroll
      for (int w = 0; w < WPT; ++w)
#pragma unroll
        for (int k = 0; k < 20; ++k) t[k] += red[wave + w][k];
      float* dH = grad_H + tok * 16;
      float* dp = grad_hp + tok * 4;
#pragma unroll
      for (int k = 0; k < 16; ++k) dH[k] = t[k];
#pragma unroll
      for (int i = 0; i < 4; ++i) dp[i] = t[16 + i];
    }
  } else if (sub == 0) {
    float* dH = grad_H + tok * 16;
    float* dp = grad_hp + tok * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      dp[i] = shp[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) dH[i * 4 + j] = sH[i][j];
    }
  }
}

int launch_k4_fwd(const uint16_t* x, const uint16_t* lo, const float* H, const float* hp,
                  uint16_t* out, int64_t T, int C, hipStream_t s) {
  with_row_walk(C, aligned16(x) && aligned16(lo) && aligned16(out), [&](auto w) {
    constexpr int L = decltype(w)::LPT;
    // Tokens narrower than a wave are faster in the loop's schedule (T = 65536,
    // C = 176 42.7 -> 36.5 us, 256 50.5 -> 48.6); wider ones equal or slower.
    using Walk = RowWalk<L, decltype(w)::LOOP || L < kWave, decltype(w)::WHOLE>;
    // Residency cap (fmhc_common.h).
    static const unsigned own = own_lds(reinterpret_cast<const void*>(&k4_fwd_kernel<Walk>));
    for_launches(T, block_of<L>(), tokens_per_block(L), [&](int64_t t, int64_t n) {
      const dim3 grid(blocks_for(n, tokens_per_block(L)));
      unsigned lds = 0;
      if (decltype(w)::LOOP)
        lds = grid.x >= kCapMinBlocks ? kLdsCapFive : 0u;
      else
        lds = cap_lds(own, grid.x, block_of<L>(), L, C / 8, Walk::CAP);
      k4_fwd_kernel<Walk><<<grid, block_of<L>(), FMHC_LDS_CAP ? lds : 0u, s>>>(
          x + t * 4 * C, lo + t * C, H + t * 16, hp + t * 4, out + t * 4 * C, n, C);
    });
  });
  return launch_status();
}

int launch_k4_fwd_pack8(const uint16_t* x, const uint16_t* lo, const float* H, const float* hp, uint16_t* out,
                        int8_t* xq, uint8_t* xs, int8_t* lq, uint8_t* ls, int64_t T, int C, hipStream_t s,
                        const uint16_t* res = nullptr) {
  // (A null xq or res counts as aligned.)
  const bool aligned = C % 8 == 0 && aligned16(x) && aligned16(lo) && aligned16(out) && aligned16(res) &&
                       Pack8Src::aligned(xq) && Pack8Src::aligned(lq);
  const int G = pack_groups(C);
  // Lanes for whole groups of 32 columns.
  auto run = [&](auto w, auto few) {
    using Walk = decltype(w);
    constexpr int L = Walk::LPT;
    auto launch = [&](auto packx, auto add) {
      constexpr bool PX = decltype(packx)::value, RES = decltype(add)::value;
      for_launches(T, block_of<L>(), tokens_per_block(L), [&](int64_t t, int64_t n) {
        const dim3 grid(blocks_for(n, tokens_per_block(L)));
        k4_fwd_pack8_kernel<Walk, decltype(few)::value, PX, RES><<<grid, block_of<L>(), 0, s>>>(
            x + t * 4 * C, lo + t * C, H + t * 16, hp + t * 4, out + t * 4 * C, PX ? xq + t * 4 * C : nullptr,
            PX ? xs + t * 4 * G : nullptr, lq + t * C, ls + t * G, n, C, RES ? res + t * C : nullptr);
      });
    };
    if (!xq)
      launch(std::false_type{}, std::false_type{});
    else
      res ? launch(std::true_type{}, std::true_type{}) : launch(std::true_type{}, std::false_type{});
  };
  if (C < 8)
    run(RowWalk<8, false, false>{}, std::true_type{});
  else
    with_row_walk(G * kPackGroup, aligned, [&](auto w) { run(w, std::false_type{}); });
  return launch_status();
}

constexpr int64_t kK4EarlyLanes = int64_t{16384} * 64;

template <typename SRC>
int launch_k4_bwd(const typename SRC::Elem* x, const typename SRC::Elem* lo, const float* H, const float* hp,
                  const uint16_t* go, uint16_t* gx, uint16_t* glo, float* gH, float* ghp,
                  int64_t T, int C, hipStream_t s, const uint8_t* xs = nullptr, const uint8_t* los = nullptr) {
  const bool aligned = SRC::aligned(x) && SRC::aligned(lo) && aligned16(go) && aligned16(gx) && aligned16(glo);
  with_row_walk(C, aligned, [&](auto w) {
    using Walk = decltype(w);
    constexpr int L = Walk::LPT;
    auto launch = [&](auto walk, auto early) {
      using W = decltype(walk);
      constexpr bool E = decltype(early)::value;
      // Residency cap (fmhc_common.h) with one group per lane, up to 256 lanes
      // (T = 30000, C = 3000 440 us with and without).
      static const unsigned own = own_lds(reinterpret_cast<const void*>(&k4_bwd_kernel<W, E, SRC>));
      for_launches(T, block_of<L>(), tokens_per_block(L), [&](int64_t t, int64_t n) {
        const dim3 grid(blocks_for(n, tokens_per_block(L)));
        unsigned lds = 0;
        if (FMHC_LDS_CAP && C / 8 <= L && L <= 256) lds = cap_lds(own, grid.x, block_of<L>(), L, C / 8, Walk::CAP);
        k4_bwd_kernel<W, E, SRC><<<grid, block_of<L>(), lds, s>>>(
            x + t * 4 * C, lo + t * C, H + t * 16, hp + t * 4, go + t * 4 * C, gx + t * 4 * C, glo + t * C,
            gH + t * 16, ghp + t * 4, n, C, SRC::kPacked ? xs + t * 4 * pack_groups(C) : nullptr,
            SRC::kPacked ? los + t * pack_groups(C) : nullptr);
      });
    };
    // EARLY: all of a lane's loads go out before its first store, so a wave
    // waits for one round trip instead of five, but holds more registers and
    // leaves its stores to the end.  Few waves (up to 64 per CU) and unaligned
    // rows take it (T = 1000, C = 2560 15.6 us, in the plain order 16.4; T = 1024,
    // C = 1024 8.1 / 8.3; T = 30011, C = 1001 151 / 157); many waves are faster
    // in the plain order, as the loop over groups schedules it even for one
    // group per lane (T = 65536, C = 1000 322 -> 307 us, 1024 304 -> 299, 2048
    // 618 -> 599; T = 65537, C = 2560 765 -> 756).  Tokens narrower than a wave
    // keep the coefficients in vector registers and the plain order.
    if constexpr (L < kWave)
      launch(w, std::false_type{});
    else if (!Walk::WHOLE || T * L <= kK4EarlyLanes)
      launch(w, std::true_type{});
    else
      launch(RowWalk<L, true, Walk::WHOLE>{}, std::false_type{});
  });
  return launch_status();
}

bool bad_sizes(int64_t T, int64_t C, int64_t n) {
  return T < 0 || C <= 0 || C > (int64_t{1} << 30) || n != 4;
}

}  // namespace
}  // namespace fmhc

extern "C" int fmhc_k4_fwd(const uint16_t* x, const uint16_t* lo, const float* H,
                           const float* h_post, uint16_t* out, int64_t T, int64_t C, int64_t n,
                           void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C, n)) return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (!x || !lo || !H || !h_post || !out) return FMHC_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return launch_k4_fwd(x, lo, H, h_post, out, T, static_cast<int>(C), s);
}

extern "C" int fmhc_k4_bwd(const uint16_t* x, const uint16_t* lo, const float* H,
                           const float* h_post, const uint16_t* grad_out, uint16_t* grad_x,
                           uint16_t* grad_lo, float* grad_H, float* grad_h_post, int64_t T,
                           int64_t C, int64_t n, void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C, n)) return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (!x || !lo || !H || !h_post || !grad_out || !grad_x || !grad_lo || !grad_H || !grad_h_post)
    return FMHC_ERR_INVALID_ARGUMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return launch_k4_bwd<Bf16Src>(x, lo, H, h_post, grad_out, grad_x, grad_lo, grad_H, grad_h_post, T, static_cast<int>(C),
                       s);
}

extern "C" int fmhc_k4_bwd_pack8(const int8_t* x_codes, const uint8_t* x_scales, const int8_t* lo_codes,
                                 const uint8_t* lo_scales, const float* H, const float* h_post,
                                 const uint16_t* grad_out, uint16_t* grad_x, uint16_t* grad_lo, float* grad_H,
                                 float* grad_h_post, int64_t T, int64_t C, int64_t n, void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C, n)) return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (!x_codes || !x_scales || !lo_codes || !lo_scales || !H || !h_post || !grad_out || !grad_x || !grad_lo ||
      !grad_H || !grad_h_post)
    return FMHC_ERR_INVALID_ARGUMENT;
  return launch_k4_bwd<Pack8Src>(x_codes, lo_codes, H, h_post, grad_out, grad_x, grad_lo, grad_H, grad_h_post, T,
                                 static_cast<int>(C), static_cast<hipStream_t>(stream), x_scales, lo_scales);
}

extern "C" int fmhc_k4_fwd_pack8(const uint16_t* x, const uint16_t* lo, const float* H, const float* h_post,
                                 uint16_t* out, int8_t* x_codes, uint8_t* x_scales, int8_t* lo_codes,
                                 uint8_t* lo_scales, int64_t T, int64_t C, int64_t n, void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C, n)) return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (!x || !lo || !H || !h_post || !out || !x_codes != !x_scales || !lo_codes || !lo_scales)
    return FMHC_ERR_INVALID_ARGUMENT;
  return launch_k4_fwd_pack8(x, lo, H, h_post, out, x_codes, x_scales, lo_codes, lo_scales, T, static_cast<int>(C),
                             static_cast<hipStream_t>(stream));
}

extern "C" int fmhc_k4_fwd_pack8_residual(const uint16_t* x, const uint16_t* lo, const uint16_t* residual,
                                          const float* H, const float* h_post, uint16_t* out, int8_t* x_codes,
                                          uint8_t* x_scales, int8_t* lo_codes, uint8_t* lo_scales, int64_t T, int64_t C,
                                          int64_t n, void* stream) {
  using namespace fmhc;
  if (bad_sizes(T, C, n)) return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (!x || !lo || !residual || !H || !h_post || !out || !x_codes || !x_scales || !lo_codes || !lo_scales)
    return FMHC_ERR_INVALID_ARGUMENT;
  return launch_k4_fwd_pack8(x, lo, H, h_post, out, x_codes, x_scales, lo_codes, lo_scales, T, static_cast<int>(C),
                             static_cast<hipStream_t>(stream), residual);
}
