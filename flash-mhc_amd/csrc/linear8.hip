// Products of rows in 8 bits (pack8_rows): the C entry point and its kernels.
//
//   out[t, n] = round(sum_k x[t, k] w[n, k] * x_scale[t] * w_scale[n] + bias[n] + residual[t, n])
//
// The sum is of integers and exact: |code| <= 128 and K < 2^17 keep it below 2^31.
// It is widened to fp32 (one rounding), scaled, and the output rounded once.  A token's scale past 2^96
// multiplies last (l8_value), so that only a product that is itself past fp32's range becomes infinite.
//
// Many tokens are bound by the matrix cores at the clock that the power limit leaves them: T = 16384,
// N = K = 4096 takes 209 to 218 us by card, 2.5 to 2.6 POP/s (PyTorch's integer product 269 us), where
// instructions that only read LDS reach 3.1 to 3.4 POP/s.  At K = 1024 the tiles' results take as long as their
// products' last third (T = 65536, N = 1024 72 to 73 us, 1.9 POP/s; with a residual 92 to 93).  Few tokens are
// bound by latency: T = 1, N = K = 4096 5.2 us for 16.8 MB of weight.
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
  bool lines;        // rows of out begin at multiples of 16 bytes
  int64_t T;
  int N, K;
};

constexpr int kChunk = 16;  // bytes that a lane moves
constexpr int kXcds = 8;
constexpr int kCus = 256;

// A kernel's bounds: a row is read to the next whole chunk.
__host__ __device__ __forceinline__ int l8_row_bytes(int K) { return (K + kChunk - 1) / kChunk * kChunk; }

// Bits of a dword that hold columns below n (of its four).
__device__ __forceinline__ int l8_mask(int n) { return n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1; }

// What scales a product and is added to it, for eight channels from c on (those past N as the last one).
template <int DT>
struct L8Channels {
  float s[8], b[8];
  __device__ __forceinline__ L8Channels(const L8Args& a, int c) {
    using S = typename Elems<DT>::S;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int n = c + e < a.N ? c + e : a.N - 1;
      s[e] = a.ws[n];
      b[e] = 0.f;
      if (a.bias)
        b[e] = a.bias_f32 ? static_cast<const float*>(a.bias)[n] : Elems<DT>::load(static_cast<const S*>(a.bias) + n);
    }
  }
};

// Eight elements of the residual as loaded.
template <int DT>
struct L8Raw {
  u32x4 a;
  template <bool NT>
  __device__ __forceinline__ void load(const typename Elems<DT>::S* p) {
    a = NT ? ld16_stream(p) : ld16(p);
  }
  __device__ __forceinline__ void add_to(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == FMHC_DTYPE_BF16) {
        v[2 * i] += bf_lo(a[i]);
        v[2 * i + 1] += bf_hi(a[i]);
      } else {
        v[2 * i] += Elems<DT>::widen(a[i] & 0xffffu);
        v[2 * i + 1] += Elems<DT>::widen(a[i] >> 16);
      }
    }
  }
};
template <>
struct L8Raw<FMHC_DTYPE_F32> {
  u32x4 a, b;
  template <bool NT>
  __device__ __forceinline__ void load(const float* p) {
    a = ld16(p);
    b = ld16(p + 4);
  }
  __device__ __forceinline__ void add_to(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] += __uint_as_float(a[i]);
      v[4 + i] += __uint_as_float(b[i]);
    }
  }
};

// Token scales up to this one multiply a sum (at most 2^31) within fp32's range.  Past it the channel's scale
// multiplies first: then what is on the way passes the range only where the result does.  (Scales of packed
// rows are 2^-107 or more: no product on the way is subnormal where they are.)
constexpr float kL8Large = 0x1p96f;

__device__ __forceinline__ float l8_value(int acc, float xs, float ws, float b) {
  const bool last = fabsf(xs) > kL8Large;
  return __builtin_fmaf(static_cast<float>(acc) * (last ? ws : xs), last ? xs : ws, b);
}

// Products of a token with eight channels, scaled, and the bias; ANY: the token's scale may be past kL8Large.
template <int DT, bool ANY>
__device__ __forceinline__ void l8_scale(const int (&acc)[8], const L8Channels<DT>& ch, float xs, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (ANY)
      v[e] = l8_value(acc[e], xs, ch.s[e], ch.b[e]);
    else
      v[e] = __builtin_fmaf(static_cast<float>(acc[e]) * xs, ch.s[e], ch.b[e]);
  }
}

// What a wave's lanes have written to LDS is there for its other lanes, and what they have read may be
// written over (in order by themselves; the compiler has to know).
__device__ __forceinline__ void l8_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---------------------------------------------------------------------------
// Tiles of tokens x channels through LDS.

// Waits until N vector memory instructions of the wave are under way at most.
template <int N>
__device__ __forceinline__ void l8_wait_vm() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0f70);
}

// BT tokens x BC channels per workgroup, WT x WC waves, steps of BK columns, NB (2 or 4) of them in LDS.
template <int kBT, int kBC, int kWT, int kWC, int kNB>
struct L8Tile {
  static constexpr int BT = kBT, BC = kBC, WT = kWT, WC = kWC, BK = 128, NB = kNB;
  static constexpr int THREADS = kWave * WT * WC;
  static constexpr int LDS = NB * (BT + BC) * BK;
};

// How a launch's workgroups walk the tiles: each XCD (workgroup id mod 8) has a run of them, in which
// eight token tiles take turns before the channel tile moves on, so that an XCD's L2 holds what its
// CUs read at a time.
struct L8Walk {
  int tiles, tiles_t, tiles_c;
  __device__ __forceinline__ int first(int id) const { return id / kXcds; }
  __device__ __forceinline__ int run(int id) const {  // tiles of this workgroup's XCD
    return tiles / kXcds + (id % kXcds < tiles % kXcds ? 1 : 0);
  }
  __device__ __forceinline__ int step(int id, int groups) const {  // workgroups of this XCD
    return groups / kXcds + (id % kXcds < groups % kXcds ? 1 : 0);
  }
  __device__ __forceinline__ void at(int id, int pos, int& t, int& c) const {
    const int xcd = id % kXcds, rest = tiles % kXcds;
    const int n = xcd * (tiles / kXcds) + (xcd < rest ? xcd : rest) + pos;
    constexpr int kGroup = 8;
    const int per = kGroup * tiles_c, g = n / per, in = n % per;
    const int rows = tiles_t - g * kGroup < kGroup ? tiles_t - g * kGroup : kGroup;
    t = __builtin_amdgcn_readfirstlane(g * kGroup + in % rows);
    c = __builtin_amdgcn_readfirstlane(in / rows);
  }
};

// A wave has up to 128 x 64 of a tile: 12 reads of LDS for 32 instructions, accumulators in half of its
// registers.  Measured in turn with the kernel as it was then, and slower (POP/s at T = N = K = 8192, against
// 2.41): 128 x 128 per wave with four waves 2.0 to 2.16, instructions of 32 x 32 x 32 2.25, four steps of 64
// columns 2.28; two workgroups of 128 x 256 in steps of 64 on a CU, so that one stores while the other
// multiplies, 79 -> 84 us at T = 65536, N = K = 1024 and 214 -> 260 at T = 16384, N = K = 4096.
//
// Loads go from memory to LDS without registers (rows of BK bytes, 16 bytes a lane), NB - 1 steps and a
// part ahead of the products, fragments from LDS to registers one part of 64 columns ahead.  The loads run on
// into the workgroup's next tile while this one's results are stored.
template <int DT, typename Tile>
__global__ __launch_bounds__(Tile::THREADS, 2) void l8_tile_kernel(const L8Args a, const L8Walk walk) {
// (The host's pass has no type for a buffer's descriptor.)
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BT = Tile::BT, BC = Tile::BC, WT = Tile::WT, WC = Tile::WC, BK = Tile::BK, NB = Tile::NB;
  constexpr int WAVES = WT * WC, MT = BT / WT / 16, MC = BC / WC / 16;
  constexpr int RPL = kWave * kChunk / BK;                     // rows per load of a wave
  constexpr int LT = BT / RPL / WAVES, LC = BC / RPL / WAVES;  // loads per wave and step
  constexpr int PARTS = BK / 64;                               // of a step: one instruction's columns
  static_assert((NB == 2 || NB == 4) && LT >= 1 && LC >= 1 && MT >= 1 && MC >= 2 && MC % 2 == 0 && PARTS % 2 == 0);
  // (Arrays of their own: in one array the compiler would wait for all loads before each read.)
  constexpr bool FOUR = NB == 4;
  __shared__ __align__(16) int8_t x0[BT * BK];
  __shared__ __align__(16) int8_t x1[BT * BK];
  __shared__ __align__(16) int8_t x2[FOUR ? BT * BK : 16];
  __shared__ __align__(16) int8_t x3[FOUR ? BT * BK : 16];
  __shared__ __align__(16) int8_t w0[BC * BK];
  __shared__ __align__(16) int8_t w1[BC * BK];
  __shared__ __align__(16) int8_t w2[FOUR ? BC * BK : 16];
  __shared__ __align__(16) int8_t w3[FOUR ? BC * BK : 16];
  __shared__ __align__(16) int turn[WAVES][16 * 16 * MC];
  using Lds = __attribute__((address_space(3))) int8_t;
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int id = static_cast<int>(blockIdx.x), run = walk.run(id), stride = walk.step(id, static_cast<int>(gridDim.x));
  // NB steps, one per buffer, at a time.
  const int bytes = l8_row_bytes(a.K), steps = (a.K + NB * BK - 1) / (NB * BK) * NB;

  // What is loaded next: rows from xp and wp on, xn and wn bytes of which can be read.  Reads past a
  // tile's last row give zeros, and so do those past the last tile.
  int xn = 0, wn = 0;
  const int8_t *xp = a.x, *wp = a.w;
  auto tile_rows = [&](int pos) __attribute__((always_inline)) {
    int t, c;
    walk.at(id, pos < run ? pos : 0, t, c);
    const int64_t t0 = static_cast<int64_t>(t) * BT, c0 = static_cast<int64_t>(c) * BC;
    const int rt = static_cast<int>(a.T - t0 < BT ? a.T - t0 : BT), rc = static_cast<int>(a.N - c0 < BC ? a.N - c0 : BC);
    xp = a.x + t0 * a.ldx;
    wp = a.w + c0 * a.ldw;
    xn = pos < run ? (rt - 1) * static_cast<int>(a.ldx) + bytes : 0;
    wn = pos < run ? (rc - 1) * static_cast<int>(a.ldw) + bytes : 0;
  };
  auto next_step = [&]() __attribute__((always_inline)) {
    xp += BK;
    wp += BK;
    xn = xn > BK ? xn - BK : 0;
    wn = wn > BK ? wn - BK : 0;
  };
  // A row's chunk j lies at j ^ (row & 7): 16 rows' same chunks spread over the banks.
  const int lrow = lane / (BK / kChunk), lchunk = lane % (BK / kChunk) ^ (RPL * wave + lrow & 7);
  int xo[LT], wo[LC];
#pragma unroll
  for (int j = 0; j < LT; ++j) xo[j] = (lrow + RPL * (wave + WAVES * j)) * static_cast<int>(a.ldx) + lchunk * kChunk;
#pragma unroll
  for (int j = 0; j < LC; ++j) wo[j] = (lrow + RPL * (wave + WAVES * j)) * static_cast<int>(a.ldw) + lchunk * kChunk;
  // Loads j0 .. j1 of a step: x's first, then w's.
  auto load = [&](int8_t* xb, int8_t* wb, int j0, int j1) __attribute__((always_inline)) {
    // (Uniform as they are; the compiler is told, or it loops over the lanes.)
    const auto xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(xp), 0, __builtin_amdgcn_readfirstlane(xn), 0x00027000);
    const auto wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(wp), 0, __builtin_amdgcn_readfirstlane(wn), 0x00027000);
#pragma unroll
    for (int j = j0; j < j1; ++j) {
      int8_t* to = (j < LT ? xb : wb) + (wave + WAVES * (j < LT ? j : j - LT)) * RPL * BK;
      if (j < LT)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (Lds*)to, kChunk, xo[j], 0, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (Lds*)to, kChunk, wo[j - LT], 0, 0, 0);
    }
  };

  const int wt = wave / WC * (BT / WT), wc = wave % WC * (BC / WC);
  const int fr = lane & 15, fk = lane >> 4;
  auto at = [&](int part) __attribute__((always_inline)) { return fr * BK + ((fk + 4 * part) ^ (fr & 7)) * kChunk; };
  // AHEAD fragments of x are in registers at a time.
  constexpr int AHEAD = MT < 4 ? MT : 4;
  i32x4 acc[MT][MC], xf[AHEAD], wf[2][MC];
  auto read_w = [&](const int8_t* wb, int part, int q, int j) __attribute__((always_inline)) {
    wf[q][j] = *reinterpret_cast<const i32x4*>(wb + (wc + 16 * j) * BK + at(part));
  };
  auto read_x = [&](const int8_t* xb, int part, int i) __attribute__((always_inline)) {
    xf[i % AHEAD] = *reinterpret_cast<const i32x4*>(xb + (wt + 16 * i) * BK + at(part));
  };
  // A wave's own loads for the next step have landed, those for the NB - 2 after it may be under way, and its
  // reads are done; then all waves'.
  auto sync = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    constexpr int N = (NB - 2) * (LT + LC);
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0070);  // vmcnt(N) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // A step with only `left` < BK columns: the others of x are set to zero (w's may be anything).
  auto cut = [&](int8_t* xb, int left) __attribute__((always_inline)) {
    if (left >= BK) return;
    for (int i = static_cast<int>(threadIdx.x); i < BT * BK / kChunk; i += Tile::THREADS) {
      const int row = i / (BK / kChunk), n = left - (i % (BK / kChunk) ^ (row & 7)) * kChunk;
      if (n >= kChunk) continue;
      auto* p = reinterpret_cast<i32x4*>(xb + i * kChunk);
      i32x4 v = *p;
#pragma unroll
      for (int d = 0; d < 4; ++d) v[d] &= l8_mask(n - 4 * d);
      *p = v;
    }
    sync();
  };

  // A buffer's parts.  Where the last one reads on into the other buffer every wave has its fragments of
  // this buffer and the other buffer's loads have landed (`left` columns of it are x's); then this buffer
  // is free.
  auto buffer = [&](int8_t* xb, int8_t* wb, int8_t* xnext, const int8_t* wnext, int left) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      const bool last = p == PARTS - 1;
      // For each fragment of x its products, with a read of the next part's w and loads between them, then
      // the read that takes its place; in this order.
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int k = i - (MT - AHEAD);  // of the next part's first fragments
        if (last && k == 0) {
          sync();
          cut(xnext, left);
          __builtin_amdgcn_sched_barrier(0);
        }
        constexpr int NL = (LT + LC + AHEAD - 1) / AHEAD;
#pragma unroll
        for (int j = 0; j < MC; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[p & 1][j], xf[i % AHEAD], acc[i][j], 0, 0, 0);
          if (j == MC / 2 - 1 && k >= 0) {
#pragma unroll
            for (int n = k; n < MC; n += AHEAD) read_w(last ? wnext : wb, last ? 0 : p + 1, (p + 1) & 1, n);
            if (last) load(xb, wb, k * NL < LT + LC ? k * NL : LT + LC, (k + 1) * NL < LT + LC ? (k + 1) * NL : LT + LC);
          }
        }
        if (k >= 0)
          read_x(last ? xnext : xb, last ? 0 : p + 1, k);
        else
          read_x(xb, p, i + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  int pos = walk.first(id);
  tile_rows(pos);
  load(x0, w0, 0, LT + LC);
  l8_wait_vm<0>();
  sync();
  cut(x0, a.K);
  next_step();
  load(x1, w1, 0, LT + LC);
  if constexpr (FOUR) {
    next_step();
    load(x2, w2, 0, LT + LC);
    next_step();
    load(x3, w3, 0, LT + LC);
  }
#pragma unroll
  for (int j = 0; j < MC; ++j) read_w(w0, 0, 0, j);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) read_x(x0, 0, i);
  for (; pos < run; pos += stride) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < MC; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    for (int s = 0; s < steps; s += NB) {
      // NB steps ahead, or the next tile's first NB.
      const int ahead = s + NB < steps ? s + NB : 0;
      if (ahead > 0)
        next_step();
      else
        tile_rows(pos + stride);
      buffer(x0, w0, x1, w1, a.K - (s + 1) * BK);
      next_step();
      if constexpr (FOUR) {
        buffer(x1, w1, x2, w2, a.K - (s + 2) * BK);
        next_step();
        buffer(x2, w2, x3, w3, a.K - (s + 3) * BK);
        next_step();
        buffer(x3, w3, x0, w0, a.K - ahead * BK);
      } else {
        buffer(x1, w1, x0, w0, a.K - ahead * BK);
      }
    }
    // A lane has four channels of a token in each fragment; through LDS it gets eight of two tokens
    // (or of more, where the wave has fewer channels), so that stores fill lines.
    int t, c;
    walk.at(id, pos, t, c);
    constexpr int CHANNELS = 16 * MC, LPR = CHANNELS / 8, ROWS = kWave / LPR;  // lanes per token, tokens at a time
    constexpr int TURNS = 16 / ROWS;                                           // token groups of a fragment
    using S = typename Elems<DT>::S;
    int ln = lane;  // (not to be kept in registers over the loop above)
    asm volatile("" : "+v"(ln));
    const int64_t t0 = static_cast<int64_t>(t) * BT + wt, left_t = a.T - t0;
    const int c0 = c * BC + wc, col = ln % LPR * 8, row = ln / LPR;
    L8Channels<DT> ch(a, c0 + col);
    // What is inside: tokens of the wave, channels of the lane.
    constexpr int most_t = 16 * MT;
    const int tokens = static_cast<int>(left_t < most_t ? left_t : most_t);
    const int mine = a.N - c0 - col < 8 ? a.N - c0 - col : 8;
    const float* xs0 = a.xs + t0;
    float xs_most = 0.f;
#pragma unroll
    for (int k = 0; k < most_t; k += kWave) xs_most = fmaxf(xs_most, fabsf(xs0[k + ln < tokens ? k + ln : tokens - 1]));
    const bool large = __builtin_amdgcn_ballot_w64(xs_most > kL8Large) != 0;
    // (Waited for here, also where no token of the lane's is stored: not in the loop above.)
#pragma unroll
    for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(ch.s[e]), "+v"(ch.b[e]));
    int* own = turn[wave];
    auto put = [&](int i) __attribute__((always_inline)) {
      const int er = ln & 15, ek = ln >> 4;
      l8_wave_sync();
#pragma unroll
      for (int j = 0; j < MC; ++j)
        *reinterpret_cast<i32x4*>(own + er * CHANNELS + ((4 * j + ek) ^ (er & (4 * MC - 1))) * 4) = acc[i][j];
      l8_wave_sync();
    };
    auto take = [&](int r, int (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<i32x4*>(v + 4 * h) =
            *reinterpret_cast<const i32x4*>(own + r * CHANNELS + ((col / 4 + h) ^ (r & (4 * MC - 1))) * 4);
    };
    auto* out0 = static_cast<S*>(a.out) + t0 * a.N + c0;
    const auto* res0 = static_cast<const S*>(a.res) + t0 * a.N + c0;
    const uint32_t at0 = static_cast<uint32_t>(row) * static_cast<uint32_t>(a.N) + static_cast<uint32_t>(col);
    // The tokens' scales and the residual are loaded before stores that their arrival would otherwise wait
    // for.  Rows that begin at 16 bytes are stored, and the residual's loaded, with the nontemporal hint:
    // neither is read again here, and what the tiles read stays cached (with / without, us, bf16: T = 65536,
    // N = 1024, K = 512 50 / 64, K = 1024 73 / 89, with a residual 93 / 102, the hint for its loads alone 93 /
    // 102; T = 16384, N = K = 4096 218 / 224).  Other rows share lines with their neighbours' stores, which are
    // to meet in the cache.  At the edges (EDGE) tokens past the last one are read as the last one, and only what
    // is inside is stored.  Tokens with scales past kL8Large take that form too: to look at the scales costs up
    // to 1% (T = 65536, N = K = 1024 71.8 -> 72.2 us, T = 16384, N = K = 4096 212.5 -> 214.1), to choose for each
    // element in every form 2% (72.3 -> 74.1 and 210.8 -> 213.8).
    auto finish = [&](auto with, auto lines, auto edge) __attribute__((always_inline)) {
      constexpr bool RES = decltype(with)::value, LINES = decltype(lines)::value, EDGE = decltype(edge)::value;
      asm volatile("" ::: "memory");  // (its loads are its own: none is under way where it is not taken)
      const int64_t by = static_cast<int64_t>(ROWS) * a.N;
      float xs[2][TURNS];
      L8Raw<DT> r[2][RES ? TURNS : 1];
      auto fetch = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
          if constexpr (EDGE) {
            const int t = 16 * i + ROWS * u + row, tc = t < tokens ? t : tokens - 1;
            xs[i & 1][u] = xs0[tc];
            if constexpr (RES) {
              if (mine == 8) r[i & 1][u].template load<false>(res0 + static_cast<int64_t>(tc) * a.N + col);
            }
          } else {
            xs[i & 1][u] = (xs0 + 16 * i + ROWS * u)[static_cast<uint32_t>(row)];
            if constexpr (RES) r[i & 1][u].template load<LINES>(res0 + (TURNS * i + u) * by + at0);
          }
        }
      };
      fetch(0);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (EDGE && 16 * i >= tokens) continue;
        if (i + 1 < MT) fetch(i + 1);
        put(i);
#pragma unroll
        for (int u = 0; u < TURNS; ++u) {
          int q[8];
          float v[8];
          take(row + ROWS * u, q);
          l8_scale<DT, EDGE>(q, ch, xs[i & 1][u], v);
          if constexpr (EDGE) {
            if (16 * i + ROWS * u + row >= tokens) continue;
            const int64_t o = (TURNS * i + u) * by + at0;
            if (mine == 8) {
              if constexpr (RES) r[i & 1][u].add_to(v);
              Elems<DT>::template store8<false>(out0 + o, v);
            } else {
#pragma unroll
              for (int e = 0; e < 7; ++e) {
                if (e >= mine) continue;
                if constexpr (RES) v[e] += Elems<DT>::load(res0 + o + e);
                Elems<DT>::store(out0 + o + e, v[e]);
              }
            }
          } else {
            if constexpr (RES) r[i & 1][u].add_to(v);
            Elems<DT>::template store8<LINES>(out0 + (TURNS * i + u) * by + at0, v);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      // Every load has arrived, only the last stores may be under way (which the compiler does not see
      // where the paths meet; it would wait in the loop above).
      constexpr int last = EDGE ? 0 : (MT > 1 ? 2 : 1) * TURNS * (DT == FMHC_DTYPE_F32 ? 2 : 1);
      l8_wait_vm<(last < 63 ? last : 63)>();
    };
    constexpr std::true_type yes;
    constexpr std::false_type no;
    if (large || left_t < most_t || c0 + CHANNELS > a.N)
      a.res ? finish(yes, no, yes) : finish(no, no, yes);
    else if (a.lines)
      a.res ? finish(yes, yes, no) : finish(no, yes, no);
    else
      a.res ? finish(yes, no, no) : finish(no, no, no);
  }
#endif
}

template <int DT, typename Tile>
void l8_tile_launch(const L8Args& a, hipStream_t s) {
  const int64_t tt = (a.T + Tile::BT - 1) / Tile::BT, tc = (a.N + Tile::BC - 1) / Tile::BC, tiles = tt * tc;
  constexpr int per_cu = kLdsPerCu / (Tile::LDS + Tile::THREADS / kWave * 16 * Tile::BC / Tile::WC * 4);
  const int64_t most = static_cast<int64_t>(kCus) * (per_cu > 4 ? 4 : per_cu);
  const L8Walk walk{static_cast<int>(tiles), static_cast<int>(tt), static_cast<int>(tc)};
  l8_tile_kernel<DT, Tile><<<dim3(static_cast<unsigned>(tiles < most ? tiles : most)), Tile::THREADS, 0, s>>>(a, walk);
}

// ---------------------------------------------------------------------------
// Few tokens: the weight's bytes, read once per 16 MT tokens.

// A workgroup has 16 MC channels and 16 MT tokens; its waves share K, each a run of columns, straight
// from memory to registers, UNROLL loads of a row under way at a time, and their sums meet in LDS.
template <int kMT, int kMC, int kWaves, int kUnroll>
struct L8Few {
  static constexpr int MT = kMT, MC = kMC, WAVES = kWaves, UNROLL = kUnroll;
};

template <int DT, typename Few>
__global__ __launch_bounds__(kWave * Few::WAVES) void l8_few_kernel(const L8Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int MT = Few::MT, MC = Few::MC, WAVES = Few::WAVES, U = Few::UNROLL;
  __shared__ __align__(16) i32x4 sums[WAVES][MT * MC][kWave];
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int c0 = static_cast<int>(blockIdx.x) * 16 * MC;
  const int64_t t0 = static_cast<int64_t>(blockIdx.y) * 16 * MT;
  const int chunks = (a.K + 63) / 64, each = (chunks + WAVES - 1) / WAVES;
  const int first = wave * each, last = first + each < chunks ? first + each : chunks;
  // Rows past the last one are read as the last one, columns past K's last whole chunk as that chunk.
  const int8_t *xp[MT], *wp[MC];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t t = t0 + 16 * i + (lane & 15);
    xp[i] = a.x + (t < a.T ? t : a.T - 1) * a.ldx;
  }
#pragma unroll
  for (int j = 0; j < MC; ++j) {
    const int c = c0 + 16 * j + (lane & 15);
    wp[j] = a.w + static_cast<int64_t>(c < a.N ? c : a.N - 1) * a.ldw;
  }
  const int end = l8_row_bytes(a.K) - kChunk, k0 = (lane >> 4) * kChunk;
  i32x4 acc[MT][MC];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < MC; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  for (int s = first; s < last; s += U) {
    i32x4 xf[U][MT], wf[U][MC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = 64 * (s + u) + k0, k = at < end ? at : end;
#pragma unroll
      for (int j = 0; j < MC; ++j) wf[u][j] = *reinterpret_cast<const i32x4*>(wp[j] + k);
#pragma unroll
      for (int i = 0; i < MT; ++i) xf[u][i] = *reinterpret_cast<const i32x4*>(xp[i] + k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= last) break;
      const int left = a.K - 64 * (s + u);  // (x's columns from K on count as zero)
      if (left < 64) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int m = l8_mask(left - k0 - 4 * d);
#pragma unroll
          for (int i = 0; i < MT; ++i) xf[u][i][d] &= m;
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < MC; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][j], xf[u][i], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < MC; ++j) sums[wave][i * MC + j][lane] = acc[i][j];
  __syncthreads();
  using S = typename Elems<DT>::S;
  constexpr int CHANNELS = 16 * MC;
  for (int o = static_cast<int>(threadIdx.x); o < 16 * MT * CHANNELS; o += kWave * WAVES) {
    const int e = o % CHANNELS, r = o / CHANNELS, c = c0 + e;
    const int64_t t = t0 + r;
    if (c >= a.N || t >= a.T) continue;
    const int* p = reinterpret_cast<const int*>(&sums[0][(r >> 4) * MC + (e >> 4)][(e >> 2 & 3) * 16 + (r & 15)]) + (e & 3);
    int v = p[0];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) v += p[k * MT * MC * kWave * 4];
    float b = 0.f;
    if (a.bias) b = a.bias_f32 ? static_cast<const float*>(a.bias)[c] : Elems<DT>::load(static_cast<const S*>(a.bias) + c);
    float y = l8_value(v, a.xs[t], a.ws[c], b);
    if (a.res) y += Elems<DT>::load(static_cast<const S*>(a.res) + t * a.N + c);
    Elems<DT>::store(static_cast<S*>(a.out) + t * a.N + c, y);
  }
#endif
}

template <int DT, typename Few>
void l8_few_launch(const L8Args& a, hipStream_t s) {
  const dim3 grid(blocks_for(a.N, 16 * Few::MC), blocks_for(a.T, 16 * Few::MT));
  l8_few_kernel<DT, Few><<<grid, kWave * Few::WAVES, 0, s>>>(a);
}

// The shortest of the tile kernels for the tiles that a product has of each, in hundredths of a round of
// 256 x 256 tiles, one per CU (52 us at K = 4096, bf16 without a residual, where all of this was measured; 43
// where there is one round).  Two of the others share a CU (a round of 512: 128 x 128 32 us, 64 x 64 13), or have
// one each (21 and 10).
struct L8Cost {
  int tile, per_cu, round, one_each;
  int64_t tiles(int64_t T, int64_t N) const { return ((T + tile - 1) / tile) * ((N + tile - 1) / tile); }
  int64_t of(int64_t T, int64_t N) const {
    const int64_t n = tiles(T, N), slots = int64_t{kCus} * per_cu;
    return n <= kCus ? one_each : (n + slots - 1) / slots * round;
  }
};
constexpr L8Cost kL8Cost256{256, 1, 100, 83}, kL8Cost128{128, 2, 62, 40}, kL8Cost64{64, 2, 25, 19};

// Without LDS where every workgroup has a CU of its own, 16 tokens each, else 32 (us, against 64 x 64 tiles:
// T = 1, N = K = 4096 5.0, 9.1; T = 64, N = 1024, K = 4096 5.8, 8.2; T = 32, N = K = 4096 8.0, 9.0, 16 tokens
// 9.5), and up to 8 tokens also where two workgroups share one (N = K = 8192: T = 1 12.7, 14.6, T = 8 14.1,
// 14.5, T = 16 16.7, 14.6).  Beyond that tiles read the operands less often (T = 64, N = K = 4096 9.3, 32
// tokens 13.4; T = 1, N = 11008, K = 4096 9.6, 10.2).
template <int DT>
int l8_run(const L8Args& a, hipStream_t s) {
  const int64_t channels = (a.N + 15) / 16;
  if ((a.T + 15) / 16 * channels <= (a.T <= 8 ? 2 : 1) * kCus) {
    l8_few_launch<DT, L8Few<1, 1, 8, 2>>(a, s);
  } else if ((a.T + 31) / 32 * channels <= kCus) {
    l8_few_launch<DT, L8Few<2, 1, 8, 2>>(a, s);
  } else {
    const int64_t large = kL8Cost256.of(a.T, a.N), medium = kL8Cost128.of(a.T, a.N), small = kL8Cost64.of(a.T, a.N);
    // Four steps in LDS where a tile has its CU alone, two where two tiles share it (128 x 128, four and two,
    // us at N = K = 4096: T = 1024 20.8, 25.8; T = 2048 37.6, 33.3); four in 64 x 64, two of which fit
    // (with two steps of 256 columns T = 128 9.4, 12.9).
    if (large <= medium && large <= small)
      l8_tile_launch<DT, L8Tile<256, 256, 2, 4, 2>>(a, s);
    else if (small < medium)
      l8_tile_launch<DT, L8Tile<64, 64, 2, 2, 4>>(a, s);
    else if (kL8Cost128.tiles(a.T, a.N) <= kCus)
      l8_tile_launch<DT, L8Tile<128, 128, 2, 2, 4>>(a, s);
    else
      l8_tile_launch<DT, L8Tile<128, 128, 2, 2, 2>>(a, s);
  }
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
  if (T < 0 || N <= 0 || K <= 0 || K >= (1 << 17) || N >= (1 << 22) || T >= (int64_t{1} << 31) || T > (int64_t{1} << 40) / N ||
      (bias_dtype != FMHC_DTYPE_F32 && bias_dtype != dtype))
    return FMHC_ERR_INVALID_ARGUMENT;
  if (dtype != FMHC_DTYPE_F32 && dtype != FMHC_DTYPE_BF16 && dtype != FMHC_DTYPE_F16) return FMHC_ERR_INVALID_ARGUMENT;
  if (T == 0) return FMHC_OK;
  if (bad_rows(x, ldx, K) || bad_rows(w, ldw, K) || !x_scales || !w_scales || !out) return FMHC_ERR_INVALID_ARGUMENT;
  const L8Args a{x, ldx, x_scales, w, ldw, w_scales, bias, bias_dtype == FMHC_DTYPE_F32, residual, out,
                 aligned16(out) && N % 8 == 0, T, static_cast<int>(N), static_cast<int>(K)};
  return with_dtype(dtype, [&](auto dt) { return l8_run<decltype(dt)::value>(a, static_cast<hipStream_t>(stream)); });
}
