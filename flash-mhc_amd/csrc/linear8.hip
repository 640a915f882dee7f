// Products of rows in 8 bits (pack8_rows): the C entry point and its kernels.
//
//   out[t, n] = round(sum_k x[t, k] w[n, k] * x_scale[t] * w_scale[n] + bias[n] + residual[t, n])
//
// The sum is of integers and exact: |code| <= 128 and K < 2^17 keep it below 2^31.
// It is widened to fp32 (one rounding), scaled, and the output rounded once.
#include "elems.h"

namespace fmhc {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct L8Args {
  const int8_t* x;
  int64_t ldx;  // bytes between rows of x
  const float* xs;
  const int8_t* w;
  int64_t ldw;
  const float* ws;
  const void* bias;  // may be null
  bool bias_f32;     // bias in fp32, otherwise in out's type
  const void* res;   // may be null
  void* out;
  int64_t T;
  int N, K;
};

constexpr int kStepK = 128;      // bytes of a row per step: two matrix instructions' k
constexpr int kChunk = 16;       // bytes that a lane moves

using Lds = __attribute__((address_space(3))) int8_t;

// (The host's pass has no type for a buffer's descriptor.)
#if defined(__HIP_DEVICE_COMPILE__)
// A tile's rows, `rows` of them in the tensor, read to a whole chunk past the row's K columns;
// reads past the last one give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t l8_rows(const int8_t* p, int64_t ld, int rows, int K) {
  const int bytes = static_cast<int>((rows - 1) * ld) + (K + kChunk - 1) / kChunk * kChunk;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(p), 0, bytes, 0x00027000);
}
#endif

// Bits of a dword that hold columns below n (of its four).
__device__ __forceinline__ int l8_mask(int n) { return n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1; }

// BT tokens x BC channels by WT x WC waves, each of which has MT x MC fragments of 16 x 16.
template <int DT, int BT, int BC, int WT, int WC>
__global__ __launch_bounds__(64 * WT * WC) void l8_tile_kernel(const L8Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int WAVES = WT * WC, MT = BT / WT / 16, MC = BC / WC / 16;
  constexpr int LT = BT / 8 / WAVES, LC = BC / 8 / WAVES;  // loads of eight rows per wave and step
  __shared__ __align__(16) int8_t xl[2][BT * kStepK];
  __shared__ __align__(16) int8_t wl[2][BC * kStepK];
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int64_t t0 = static_cast<int64_t>(blockIdx.y) * BT;
  const int c0 = static_cast<int>(blockIdx.x) * BC;
  const int rows_t = static_cast<int>(a.T - t0 < BT ? a.T - t0 : BT), rows_c = a.N - c0 < BC ? a.N - c0 : BC;
  const auto xr = l8_rows(a.x + t0 * a.ldx, a.ldx, rows_t, a.K);
  const auto wr = l8_rows(a.w + c0 * a.ldw, a.ldw, rows_c, a.K);

  // A row's chunk j lies at j ^ (row & 7): eight rows' same chunks in eight places.
  const int row0 = 8 * wave + (lane >> 3), chunk = (lane & 7) ^ (lane >> 3);
  int xo[LT], wo[LC];
#pragma unroll
  for (int j = 0; j < LT; ++j) xo[j] = (row0 + 8 * WAVES * j) * static_cast<int>(a.ldx) + chunk * kChunk;
#pragma unroll
  for (int j = 0; j < LC; ++j) wo[j] = (row0 + 8 * WAVES * j) * static_cast<int>(a.ldw) + chunk * kChunk;
  auto load = [&](int buf) {
#pragma unroll
    for (int j = 0; j < LT; ++j) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (Lds*)(xl[buf] + (wave + WAVES * j) * 8 * kStepK), 16, xo[j], 0, 0, 0);
      xo[j] += kStepK;
    }
#pragma unroll
    for (int j = 0; j < LC; ++j) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (Lds*)(wl[buf] + (wave + WAVES * j) * 8 * kStepK), 16, wo[j], 0, 0, 0);
      wo[j] += kStepK;
    }
  };

  const int wt = wave / WC * (BT / WT), wc = wave % WC * (BC / WC);
  i32x4 acc[MT][MC];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < MC; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

  const int steps = (a.K + kStepK - 1) / kStepK;
  load(0);
  for (int k = 0; k < steps; ++k) {
    __syncthreads();
    if (k + 1 < steps) load((k + 1) & 1);
    const int8_t* xb = xl[k & 1];
    const int8_t* wb = wl[k & 1];
    const int left = a.K - k * kStepK;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = (lane >> 4) + 4 * h;
      const int at = (lane & 15) * kStepK + ((c ^ (lane & 7)) * kChunk);
      i32x4 xf[MT], wf[MC];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xf[i] = *reinterpret_cast<const i32x4*>(xb + (wt + 16 * i) * kStepK + at);
        if (left < kStepK) {
#pragma unroll
          for (int d = 0; d < 4; ++d) xf[i][d] &= l8_mask(left - c * kChunk - 4 * d);
        }
      }
#pragma unroll
      for (int j = 0; j < MC; ++j) wf[j] = *reinterpret_cast<const i32x4*>(wb + (wc + 16 * j) * kStepK + at);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < MC; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[i], acc[i][j], 0, 0, 0);
    }
  }

  // A lane has four channels of a token in each fragment.
  using S = typename Elems<DT>::S;
  auto* out = static_cast<S*>(a.out);
  const auto* res = static_cast<const S*>(a.res);
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t t = t0 + wt + 16 * i + (lane & 15);
    if (t >= a.T) continue;
    const float xs = a.xs[t];
#pragma unroll
    for (int j = 0; j < MC; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = c0 + wc + 16 * j + (lane >> 4) * 4 + e;
        if (c >= a.N) continue;
        float b = 0.f;
        if (a.bias) b = a.bias_f32 ? static_cast<const float*>(a.bias)[c] : Elems<DT>::load(static_cast<const S*>(a.bias) + c);
        float v = __builtin_fmaf(static_cast<float>(acc[i][j][e]) * xs, a.ws[c], b);
        if (res) v += Elems<DT>::load(res + t * a.N + c);
        Elems<DT>::store(out + t * a.N + c, v);
      }
    }
  }
#endif
}

template <int DT>
int l8_run(const L8Args& a, hipStream_t s) {
  const dim3 grid(blocks_for(a.N, 128), blocks_for(a.T, 128));
  l8_tile_kernel<DT, 128, 128, 2, 2><<<grid, 256, 0, s>>>(a);
  return launch_status();
}

// Rows that a kernel reads: whole chunks from 16-byte addresses, offsets of a tile in 31 bits.
bool bad_rows(const int8_t* p, int64_t ld, int64_t K) {
  return !p || !aligned16(p) || ld % kChunk != 0 || ld < K || ld > (int64_t{1} << 22);
}

}  // namespace

}  // namespace fmhc

extern "C" int fmhc_linear8(const int8_t* x, int64_t ldx, const float* x_scales, const int8_t* w, int64_t ldw,
                            const float* w_scales, const void* bias, const void* residual, void* out, int dtype,
                            int bias_dtype, int64_t T, int64_t N, int64_t K, void* stream) {
  using namespace fmhc;
  if (T < 0 || N <= 0 || K <= 0 || K >= (1 << 17) || N > (int64_t{1} << 30) || T > (int64_t{1} << 60) / N ||
      (bias_dtype != FMHC_DTYPE_F32 && bias_dtype != dtype))
    return FMHC_ERR_INVALID_ARGUMENT;
  if (dtype != FMHC_DTYPE_F32 && dtype != FMHC_DTYPE_BF16 && dtype != FMHC_DTYPE_F16) return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (bad_rows(x, ldx, K) || bad_rows(w, ldw, K) || !x_scales || !w_scales || !out) return FMHC_ERR_INVALID_ARGUMENT;
  const L8Args a{x, ldx, x_scales, w, ldw, w_scales, bias, bias_dtype == FMHC_DTYPE_F32, residual, out, T,
                 static_cast<int>(N), static_cast<int>(K)};
  return with_dtype(dtype, [&](auto dt) { return l8_run<decltype(dt)::value>(a, static_cast<hipStream_t>(stream)); });
}
