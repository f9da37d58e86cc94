// Rows in 8 bits times a matrix in 8 bits, with a scale for each token and
// each output channel:
//     out[m, n] = sx[m] sw[n] sum_k x[m, k] w[n, k] + bias[n].
// The sum is exact: products of at most 2^14 in int32, K <= 131071.  The
// scales, the bias and the rounding to the output's type are one fp32 step at
// the end, so the result does not depend on how the sum is cut.
#include "mrsa_device.h"

using namespace mrsa;

namespace {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

template <class E, int N>
struct __attribute__((packed, aligned(1))) Pack {
  E e[N];
};
__device__ __forceinline__ u32x4_t load16(const int8_t* p) {  // any alignment
  const Pack<uint32_t, 4> v = *reinterpret_cast<const Pack<uint32_t, 4>*>(p);
  return u32x4_t{v.e[0], v.e[1], v.e[2], v.e[3]};
}

struct LinearArgs {
  const int8_t* x;
  const int8_t* w;
  const float* sx;
  const float* sw;
  const void* bias;      // optional, of the output's type
  void* out;             // dense [M, N]
  int32_t* partial;      // parts > 1
  int64_t M, N, K, x_stride, w_stride;
  int32_t dtype, parts, tiles_m, tiles_n;
};

__device__ __forceinline__ float widen(const void* p, int64_t at, int dtype) {
  if (dtype == MRSA_DTYPE_FP32) return ((const float*)p)[at];
  const uint16_t e = ((const uint16_t*)p)[at];
  return dtype == MRSA_DTYPE_BF16 ? bf16_to_f32(e) : (float)__builtin_bit_cast(_Float16, e);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, int dtype) {
  if (dtype == MRSA_DTYPE_BF16) return pack_bf16x2(lo, hi);
  const uint32_t a = __builtin_bit_cast(uint16_t, (_Float16)lo);
  const uint32_t b = __builtin_bit_cast(uint16_t, (_Float16)hi);
  return a | b << 16;
}
__device__ __forceinline__ float scaled(int32_t sum, float sx, float sw, float bias) {
  return fmaf((float)sum * sx, sw, bias);
}

// Bytes of a row's chunk [k, k + 16): read at min(k, K - 16), and those before k (part of the
// chunk before, or all of a chunk past K) made zero in one of the two operands.
__device__ __forceinline__ u32x4_t without_first(u32x4_t v, int64_t bytes) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int n = (int)min(max(bytes - 4 * d, (int64_t)0), (int64_t)4);
    v[d] = n == 4 ? 0u : v[d] >> (8 * n) << (8 * n);
  }
  return v;
}

// ---- many rows: tiles through LDS -------------------------------------------------------

// A step is 128 bytes of K: whole cache lines.
constexpr int kStep = 128;

// WS and XS: steps of W and of X that are in LDS at once.
template <int TM_, int TN_, int WM_, int WN_, int WS_, int XS_>
struct Tile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, WS = WS_, XS = XS_;
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int MT = TM / WM / 16, NT = TN / WN / 16;   // 16 x 16 products of a wave
  static constexpr int W_SLOT = TN * kStep, X_SLOT = TM * kStep;   // bytes of a step
  static constexpr int X_LDS = WS * W_SLOT, SLOTS_END = X_LDS + XS * X_SLOT;
  static constexpr int PW = W_SLOT / 1024 / WAVES, PX = X_SLOT / 1024 / WAVES;   // 1 KB, of a wave
  static constexpr int COLS = 16 * NT;
  static constexpr int ROWS = (16 * MT + 63) / 64;             // loads of a wave's rows' scales
  static constexpr int SCALES = 2 * COLS + 64 * ROWS;           // floats, of a wave
  // One more step of W than of X: the scales have no room of their own.
  static constexpr bool SHARED = WS > XS;
  static constexpr int LDS = SLOTS_END + (SHARED ? 0 : 4 * WAVES * SCALES);
  static_assert(W_SLOT % (1024 * WAVES) == 0 && X_SLOT % (1024 * WAVES) == 0 && NT == 4 &&
                LDS <= 160 * 1024 && XS >= 2 && (WS == XS || (WS == 3 && XS == 2)) &&
                4 * WAVES * SCALES <= W_SLOT);
};

// Chunk c (16 bytes) of row r lies in place c ^ swizzle(r) of the row: the sixteen rows of a
// product's operand meet all banks.  X's are 16 consecutive ones; W's are those of column_of, so
// that a lane's results of two products are eight consecutive columns.
__device__ __forceinline__ int swizzle(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int swizzle_w(int r) { return ((r >> 1) & 1) | ((r >> 3) & 3) << 1; }
// The column of W's product nt that its operand's row r is.
__device__ __forceinline__ int column_of(int nt, int r) {
  return 32 * (nt >> 1) + 8 * (r >> 2) + 4 * (nt & 1) + (r & 3);
}

__device__ __forceinline__ u32x4_t lds16(uint32_t at) {
  return *(const __attribute__((address_space(3))) u32x4_t*)(uintptr_t)at;
}
__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
__device__ __forceinline__ i32x4_t mfma(u32x4_t a, u32x4_t b, i32x4_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a),
                                               __builtin_bit_cast(i32x4_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ const int8_t* uniform(const int8_t* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const int8_t*)(uintptr_t)((uint64_t)hi << 32 | lo);
}

// 1 KB of LDS from `to` on, lane l's 16 bytes from base + at.  As asm, since after the builtin
// the compiler waits for all DMA in flight before the next LDS read; the loop's own waits order
// them.  (s_nop: m0 and scalars that a vector instruction has just written.)
__device__ __forceinline__ void dma(uint32_t to, const int8_t* base, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %2, %1" ::"s"(
                   __builtin_amdgcn_readfirstlane(to)),
               "s"(uniform(base)), "v"(at)
               : "memory", "m0");
}

// Tiles in an order that gives each XCD (workgroups go round them) a contiguous range of bands of
// 4 tile rows, walked column by column: its concurrent tiles share operands in its L2.  (Bands of
// 8: 16384 x 3584 of 18944 values 952 us instead of 901, 16384 x 37888 of 3584 1883 instead of
// 1912; of 16: 1007 instead of 951, and 4096 x 8192 of 8192 234 instead of 224.)
__device__ __forceinline__ void tile_of(int b, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int tiles = tiles_m * tiles_n, each = tiles / 8, more = tiles % 8;
  const int xcd = b % 8, i = b / 8;
  const int t = xcd * each + min(xcd, more) + i;
  const int band = t / (4 * tiles_n), rest = t - band * 4 * tiles_n;
  const int rows = min(4, tiles_m - 4 * band);
  tn = __builtin_amdgcn_readfirstlane(rest / rows);
  tm = __builtin_amdgcn_readfirstlane(4 * band + rest - tn * rows);
}

template <class T>
struct Position {
  int lane, wave, wm, wn;
  int64_t m0, n0;  // of the tile
  __device__ __forceinline__ Position(const LinearArgs& a, int tile) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wm = wave / T::WN;
    wn = wave % T::WN;
    int tm, tn;
    tile_of(tile, a.tiles_m, a.tiles_n, tm, tn);
    m0 = (int64_t)tm * T::TM;
    n0 = (int64_t)tn * T::TN;
  }
};

// Four bytes a lane.
__device__ __forceinline__ void dma4(uint32_t to, const int8_t* base, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %2, %1" ::"s"(
                   __builtin_amdgcn_readfirstlane(to)),
               "s"(uniform(base)), "v"(at)
               : "memory", "m0");
}

template <class T>
__device__ __forceinline__ void clear(i32x4_t (&acc)[T::MT][T::NT]) {
#pragma unroll
  for (int m = 0; m < T::MT; ++m)
#pragma unroll
    for (int n = 0; n < T::NT; ++n) acc[m][n] = i32x4_t{0, 0, 0, 0};
}

// The scales (and the bias) of the wave's columns and rows, to LDS of its own: [columns], [bias],
// [rows].  By DMA, behind which the first operands are waited for anyway; a bias is loaded where
// there is one, so that nothing else depends on its type.
template <class T>
__device__ __forceinline__ void fetch_scales(const LinearArgs& a, const Position<T>& p,
                                             float* scales) {
  const int64_t n0 = min(p.n0 + p.wn * T::COLS, a.N - 1);
  const int64_t m0 = min(p.m0 + p.wm * 16 * T::MT, a.M - 1);
  const uint32_t to = lds_at(scales);
  static_assert(T::COLS == 64);
  const int64_t n = min(n0 + p.lane, a.N - 1);
  dma4(to, (const int8_t*)(a.sw + n0), 4u * (uint32_t)(n - n0));
#pragma unroll
  for (int i = 0; i < T::ROWS; ++i)
    dma4(to + 4 * (2 * T::COLS + 64 * i), (const int8_t*)(a.sx + m0),
         4u * (uint32_t)(min(m0 + 64 * i + p.lane, a.M - 1) - m0));
  scales[T::COLS + p.lane] = a.bias ? widen(a.bias, n, a.dtype) : 0.f;
}

// Eight results of row m from column n < N on.
__device__ __forceinline__ void put8(const LinearArgs& a, int64_t m, int64_t n, i32x4_t lo,
                                     i32x4_t hi, float sx, const float (&scale)[8],
                                     const float (&bias)[8]) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    y[i] = scaled(i < 4 ? lo[i & 3] : hi[i & 3], sx, scale[i], bias[i]);
  if (a.dtype == MRSA_DTYPE_FP32) {
    float* const to = (float*)a.out + m * a.N + n;
    if (n + 8 <= a.N) {
      *reinterpret_cast<Pack<float, 4>*>(to) = Pack<float, 4>{{y[0], y[1], y[2], y[3]}};
      *reinterpret_cast<Pack<float, 4>*>(to + 4) = Pack<float, 4>{{y[4], y[5], y[6], y[7]}};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < a.N) to[i] = y[i];
    }
  } else {
    uint16_t* const to = (uint16_t*)a.out + m * a.N + n;
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack2(y[2 * i], y[2 * i + 1], a.dtype);
    if (n + 8 <= a.N) {
      *reinterpret_cast<Pack<uint32_t, 4>*>(to) = Pack<uint32_t, 4>{{v[0], v[1], v[2], v[3]}};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < a.N) to[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// Sums to results.  W is the products' first operand: lane l holds, of row l % 16, columns
// 8 (l / 16) .. + 7 of two products: 16 bytes (or 32) to write, 64 bytes of a row by one
// instruction.
template <class T>
__device__ __forceinline__ void finish(const LinearArgs& a, const Position<T>& p,
                                       const float* scales, const i32x4_t (&acc)[T::MT][T::NT]) {
  constexpr int PAIRS = T::NT / 2;
  const int c0 = 8 * (p.lane >> 4);
  const int64_t n0 = p.n0 + p.wn * T::COLS + c0;
  const int64_t m0 = p.m0 + p.wm * 16 * T::MT + (p.lane & 15);
  float scale[PAIRS][8], bias[PAIRS][8];
#pragma unroll
  for (int q = 0; q < PAIRS; ++q)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4_t s = *(const f32x4_t*)(scales + 32 * q + c0 + 4 * h);
      const f32x4_t b = *(const f32x4_t*)(scales + T::COLS + 32 * q + c0 + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        scale[q][4 * h + i] = s[i];
        bias[q][4 * h + i] = b[i];
      }
    }
  float sx[T::MT];
#pragma unroll
  for (int mt = 0; mt < T::MT; ++mt) sx[mt] = scales[2 * T::COLS + 16 * mt + (p.lane & 15)];
#pragma unroll
  for (int mt = 0; mt < T::MT; ++mt) {
    const int64_t m = m0 + 16 * mt;
    if (m >= a.M) break;
#pragma unroll
    for (int q = 0; q < PAIRS; ++q) {
      const int64_t n = n0 + 32 * q;
      if (n < a.N)
        put8(a, m, n, acc[mt][2 * q], acc[mt][2 * q + 1], sx[mt], scale[q], bias[q]);
    }
  }
}

// A workgroup computes one part of K of a tile, each wave (16 MT) x 64 of it, W as the products'
// first operand.  DMA: rows 16-byte aligned and K a multiple of 16, from 128 on.  Otherwise rows go
// through registers, a step ahead.
//
// What bounds the large shapes is bringing operands from L2 to LDS: at 256 x 256 results a CU's
// registers are full, and a step's 64 KB come in where the matrix cores need 2048 cycles for its
// products.  16384 x 37888 of 3584 values take 1927 us (2310 TOPS, matrix cores 57% busy); the same
// with one row of X and W read over and over 1419, with values all zero 1900 (so not the clocks).
// Hence steps of 128 bytes (64-byte steps ask L2 twice as often: 4096 x 8192 of 8192 268 us, 223),
// three steps of W in LDS and two of X (two and two: 2022 us, since W misses L2 and X seldom does),
// and one barrier a step, between its halves, behind which reads and DMA have the second half's
// products to hide under (at the step's end: 4096 x 8192 of 8192 218 us, 212).  16 x 16 x 64
// products sustain more than 32 x 32 x 32 (random operands, nothing else running: 3966 TOPS,
// 3284).  Slower when tried: four waves of 128 x 128 (302 us against 220: a SIMD's one wave has no
// other to wait behind), a persistent workgroup with the next tile's DMA ahead of the epilogue
// (2060 us against 1989), results through LDS (4090 x 4100 of 96: 27.6 us against 22.8) or past the
// caches (2017 against 1988), W or X read as streaming data (2049, 2076 against 1979).
template <class T, bool DMA>
__global__ void __launch_bounds__(T::THREADS, T::WAVES / 4 * (T::WAVES > 4 ? 1 : 2))
    int8_tile_kernel(LinearArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[T::LDS];
  constexpr int PW = T::PW, PX = T::PX, MT = T::MT, NT = T::NT;
  const int tiles = a.tiles_m * a.tiles_n;
  const int part = blockIdx.x / tiles, tile = blockIdx.x - part * tiles;
  const int steps = (int)((a.K + kStep - 1) / kStep);
  const int tail = (int)(a.K - (int64_t)(steps - 1) * kStep);  // bytes of the last step
  const int t0 = (int)((int64_t)steps * part / a.parts);
  const int t1 = (int)((int64_t)steps * (part + 1) / a.parts);
  const Position<T> p(a, tile);
  // The scales' place.  SHARED: the slot of W that the last two steps leave free.
  float* const scales =
      (float*)(lds + (!T::SHARED ? T::SLOTS_END : (DMA ? (t1 + 1 - t0) % 3 : 2) * T::W_SLOT)) +
      p.wave * T::SCALES;
  if (a.parts == 1 && (!T::SHARED || !DMA || t1 - t0 == 1)) fetch_scales<T>(a, p, scales);
  const int lane = p.lane, wave = p.wave;

  // ---- operands in LDS: row lane % 16 of a product, chunk lane / 16 of its 64 bytes.  (Products
  // 2 i and 2 i + 1 of W: rows 32 i .., the second's four further on.)
  const uint32_t lds0 = lds_at(lds);
  uint32_t w_at[2], x_at[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int r = lane & 15, c = 4 * s + (lane >> 4), rw = column_of(0, r);
    w_at[s] = lds0 + (p.wn * T::COLS + rw) * kStep + 16u * (c ^ swizzle_w(rw));
    x_at[s] = lds0 + T::X_LDS + (p.wm * 16 * MT + r) * kStep + 16u * (c ^ swizzle(r));
  }
  auto w_read = [&](int s, int n, uint32_t slot) {
    return lds16(w_at[s] + slot + kStep * column_of(n, 0));
  };
  auto x_read = [&](int s, int m, uint32_t slot) {
    return lds16(x_at[s] + slot + 16 * kStep * m);
  };
  i32x4_t acc[MT][NT];
  clear<T>(acc);
  u32x4_t w[2][NT], x[MT];
  // The last step is the last 128 bytes of K: what the step before has, too, is made zero in W.
  auto cut = [&](u32x4_t (&f)[NT], int s) {
    const bool in = 64 * s + 16 * (lane >> 4) >= kStep - tail;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int d = 0; d < 4; ++d) f[n][d] = in ? f[n][d] : 0u;
  };
  // piece i of the wave, of W or of X: eight rows of a step
  const uint32_t w_to = lds0 + wave * PW * 1024, x_to = lds0 + T::X_LDS + wave * PX * 1024;
  auto w_row = [&](int i) { return (wave * PW + i) * 8 + (lane >> 3); };
  auto x_row = [&](int i) { return (wave * PX + i) * 8 + (lane >> 3); };
  auto w_chunk = [&](int i) { return (lane & 7) ^ swizzle_w(w_row(i)); };
  auto x_chunk = [&](int i) { return (lane & 7) ^ swizzle(x_row(i)); };

  if constexpr (DMA) {
    // Where this wave's pieces come from: rows past the end repeat the last one.
    const int8_t* const w_from = uniform(a.w + p.n0 * a.w_stride);
    const int8_t* const x_from = uniform(a.x + p.m0 * a.x_stride);
    uint32_t w_off[PW], x_off[PX];
#pragma unroll
    for (int i = 0; i < PW; ++i)
      w_off[i] = (uint32_t)(min((int64_t)w_row(i), a.N - 1 - p.n0) * a.w_stride) + 16u * w_chunk(i);
#pragma unroll
    for (int i = 0; i < PX; ++i)
      x_off[i] = (uint32_t)(min((int64_t)x_row(i), a.M - 1 - p.m0) * a.x_stride) + 16u * x_chunk(i);
    auto issue_w = [&](int t, int i, uint32_t slot) {
      dma(w_to + slot + 1024 * i, w_from + min((int64_t)t * kStep, a.K - kStep), w_off[i]);
    };
    auto issue_x = [&](int t, int i, uint32_t slot) {
      dma(x_to + slot + 1024 * i, x_from + min((int64_t)t * kStep, a.K - kStep), x_off[i]);
    };
    // The wave's own pieces of a step have landed (the LATER ones behind them may be on their
    // way), its reads are done, and so for every wave.
    auto arrived = [&](auto later) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(later()) : "memory");
    };
    constexpr int WS = T::WS, XS = T::XS;
    auto none = [] { return 0; };
    auto most = [] { return WS > XS ? PW : (PW + PX) * (XS - 2); };
    auto after = [](uint32_t slot, int slots, int bytes) {
      return slot == (uint32_t)((slots - 1) * bytes) ? 0u : slot + (uint32_t)bytes;
    };
    // Pieces in the order in which steps need them, X's ahead of W's: after those of step t come
    // at most `most` others.
#pragma unroll
    for (int j = 0; j < WS - 1; ++j) {
      if (t0 + j >= t1) break;
      if (j < XS - 1) {
#pragma unroll
        for (int i = 0; i < PX; ++i) issue_x(t0 + j, i, j * T::X_SLOT);
      }
#pragma unroll
      for (int i = 0; i < PW; ++i) issue_w(t0 + j, i, j * T::W_SLOT);
    }
    if (t0 + WS - 2 < t1) arrived(most);
    else arrived(none);
#pragma unroll
    for (int n = 0; n < NT; ++n) w[0][n] = w_read(0, n, 0);
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = x_read(0, m, 0);
    if (t0 + XS - 1 < t1) {
#pragma unroll
      for (int i = 0; i < PX; ++i) issue_x(t0 + XS - 1, i, (XS - 1) * T::X_SLOT);
    }
    if (t0 + WS - 1 < t1) {
#pragma unroll
      for (int i = 0; i < PW; ++i) issue_w(t0 + WS - 1, i, (WS - 1) * T::W_SLOT);
    }
    uint32_t w_slot = 0, x_slot = 0;
    for (int t = t0; t < t1; ++t) {
      // (in registers that the products need no copies of)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) asm volatile("" : "+v"(acc[m][n]));
      const bool partial = t == steps - 1 && tail < kStep;
      const uint32_t w_next = after(w_slot, WS, T::W_SLOT), x_next = after(x_slot, XS, T::X_SLOT);
      // first half: its products, each row tile's operand replaced by the second half's
      if (partial) cut(w[0], 0);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = mfma(w[0][n], x[m], acc[m][n]);
        constexpr int WR = (NT + MT - 1) / MT;
#pragma unroll
        for (int n = m * WR; n < (m + 1) * WR && n < NT; ++n) w[1][n] = w_read(1, n, w_slot);
        x[m] = x_read(1, m, x_slot);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (partial) cut(w[1], 1);
      // in between: the next step has arrived for every wave, and every wave has read all of this
      // one, whose slots steps WS and XS further on then fill
      if (t + WS - 1 < t1) arrived(most);
      else arrived(none);
      // second half: each row tile's operand replaced by the next step's (behind the last step:
      // read, not used)
      const bool more_w = t + WS < t1, more_x = t + XS < t1;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = mfma(w[1][n], x[m], acc[m][n]);
        constexpr int WR = (NT + MT - 1) / MT, EACH = (PX + PW + MT - 1) / MT;
#pragma unroll
        for (int n = m * WR; n < (m + 1) * WR && n < NT; ++n) w[0][n] = w_read(0, n, w_next);
        x[m] = x_read(0, m, x_next);
#pragma unroll
        for (int i = m * EACH; i < (m + 1) * EACH && i < PX + PW; ++i) {
          if (i < PX) {
            if (more_x) issue_x(t + XS, i, x_slot);
          } else {
            if (more_w) issue_w(t + WS, i - PX, w_slot);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      // (every wave has read this step, and none comes that fills its slot of W)
      if (T::SHARED && t + 2 == t1 && a.parts == 1) fetch_scales<T>(a, p, scales);
      w_slot = w_next;
      x_slot = x_next;
    }
  } else {
    // Through registers; rows at any address, K from 16 on.
    u32x4_t w_held[PW], x_held[PX];
    const int8_t *w_from[PW], *x_from[PX];
#pragma unroll
    for (int i = 0; i < PW; ++i) w_from[i] = a.w + min(p.n0 + w_row(i), a.N - 1) * a.w_stride;
#pragma unroll
    for (int i = 0; i < PX; ++i) x_from[i] = a.x + min(p.m0 + x_row(i), a.M - 1) * a.x_stride;
    auto load = [&](int t) {
      const int64_t k0 = (int64_t)t * kStep;
      if (k0 + kStep <= a.K) {
#pragma unroll
        for (int i = 0; i < PW; ++i) w_held[i] = load16(w_from[i] + k0 + 16 * w_chunk(i));
#pragma unroll
        for (int i = 0; i < PX; ++i) x_held[i] = load16(x_from[i] + k0 + 16 * x_chunk(i));
      } else {
#pragma unroll
        for (int i = 0; i < PW; ++i) {
          const int64_t k = k0 + 16 * w_chunk(i), at = min(k, a.K - 16);
          w_held[i] = without_first(load16(w_from[i] + at), k - at);
        }
#pragma unroll
        for (int i = 0; i < PX; ++i)
          x_held[i] = load16(x_from[i] + min(k0 + 16 * x_chunk(i), a.K - 16));
      }
    };
    auto store = [&](int slot) {
      auto put = [&](uint32_t at, u32x4_t v) {
        *(__attribute__((address_space(3))) u32x4_t*)(uintptr_t)(at + 16 * lane) = v;
      };
#pragma unroll
      for (int i = 0; i < PW; ++i) put(w_to + slot * T::W_SLOT + 1024 * i, w_held[i]);
#pragma unroll
      for (int i = 0; i < PX; ++i) put(x_to + slot * T::X_SLOT + 1024 * i, x_held[i]);
      __syncthreads();
    };
    load(t0);
    store(0);
    int slot = 0;
    for (int t = t0; t < t1; ++t) {
      if (t + 1 < t1) load(t + 1);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int n = 0; n < NT; ++n) w[0][n] = w_read(s, n, slot * T::W_SLOT);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          x[m] = x_read(s, m, slot * T::X_SLOT);
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[m][n] = mfma(w[0][n], x[m], acc[m][n]);
        }
      }
      slot ^= 1;
      if (t + 1 < t1) store(slot);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the scales)
  }
  if (a.parts > 1) {
    // the registers as they are, 16 bytes a lane
    i32x4_t* const to_part = (i32x4_t*)a.partial +
        ((int64_t)tile * a.parts + part) * (MT * NT * T::THREADS) + threadIdx.x;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) to_part[(m * NT + n) * T::THREADS] = acc[m][n];
    return;
  }
  finish<T>(a, p, scales, acc);
}

// Sums of a tile's parts and its results, for eight columns of a row a thread: two of the
// registers that int8_tile_kernel kept, of one of its lanes.  Bound by the partial sums' bytes from
// the caches: 1024 x 3584 in two parts 9.2 us (29 MB in, 7 MB out).
template <class T>
__global__ void __launch_bounds__(T::THREADS) int8_join_kernel(LinearArgs a) {
  constexpr int PAIRS = T::MT * T::NT / 2, EACH = 2 * PAIRS * T::THREADS;
  const int tile = blockIdx.x / PAIRS, pair = blockIdx.x - tile * PAIRS;
  const Position<T> p(a, tile);
  const i32x4_t* from = (const i32x4_t*)a.partial + (int64_t)tile * a.parts * EACH +
                        2 * pair * T::THREADS + threadIdx.x;
  i32x4_t lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
  for (int part = 0; part < a.parts; ++part, from += EACH) {
    lo += from[0];
    hi += from[T::THREADS];
  }
  const int64_t m = p.m0 + (p.wm * T::MT + pair / (T::NT / 2)) * 16 + (p.lane & 15);
  const int64_t n = p.n0 + p.wn * T::COLS + 32 * (pair % (T::NT / 2)) + 8 * (p.lane >> 4);
  if (m >= a.M || n >= a.N) return;
  float scale[8], bias[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t c = min(n + i, a.N - 1);
    scale[i] = a.sw[c];
    bias[i] = a.bias ? widen(a.bias, c, a.dtype) : 0.f;
  }
  put8(a, m, n, lo, hi, a.sx[m], scale, bias);
}

// ---- few rows: the weights' bytes ---------------------------------------------------------

// Four results of row m from column n on.
__device__ __forceinline__ void put4(const LinearArgs& a, int64_t m, int64_t n, i32x4_t sum) {
  if (m >= a.M) return;
  const float sx = a.sx[m];
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = min(n + i, a.N - 1);
    y[i] = scaled(sum[i], sx, a.sw[c], a.bias ? widen(a.bias, c, a.dtype) : 0.f);
  }
  if (a.dtype == MRSA_DTYPE_FP32) {
    float* const to = (float*)a.out + m * a.N + n;
    if (n + 4 <= a.N) {
      *reinterpret_cast<Pack<float, 4>*>(to) = Pack<float, 4>{{y[0], y[1], y[2], y[3]}};
    } else {
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) to[i] = y[i];
    }
  } else {
    uint16_t* const to = (uint16_t*)a.out + m * a.N + n;
    const uint32_t v[2] = {pack2(y[0], y[1], a.dtype), pack2(y[2], y[3], a.dtype)};
    if (n + 4 <= a.N) {
      *reinterpret_cast<Pack<uint32_t, 2>*>(to) = Pack<uint32_t, 2>{{v[0], v[1]}};
    } else {
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) to[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// Bound by W's bytes from HBM: 32 rows, 37888 x 3584 in 26.7 us (138 MB, 5.2 TB/s, a large copy's
// rate); one row, 4608 x 3584 in 5.4 us (16.5 MB, 3.1 TB/s: 144 workgroups, whose waves take seven
// steps each, two of them in flight; eight waves or deeper rings gained nothing there and cost 15%
// at 37888 columns).
//
// Consecutive lanes fetch consecutive bytes of a row, which operands loaded straight from memory
// (16 rows side by side: 60 us where this takes 31) do not.  A workgroup has 16 NT columns and up
// to 16 MT rows; its waves take K's steps of 128 in turn, each through a ring of its own in LDS,
// RING steps deep, without barriers, and add their sums in the end.  DMA: aligned rows, K from 128
// on.  Otherwise the rows go through registers, RING steps ahead, and one step of LDS.  More rows
// than 16 MT: blockIdx.y.
template <int MT, int NT, int WAVES, int RING, bool DMA>
__global__ void __launch_bounds__(64 * WAVES) int8_stream_kernel(LinearArgs a) {
  constexpr int P = 2 * NT + 2 * MT, SLOT = P * 1024, Q = MT * NT;
  constexpr int SLOTS = DMA ? RING : 1;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[WAVES * SLOTS * SLOT];
  static_assert(Q * 1024 <= SLOTS * SLOT && RING >= 2 && RING <= 4);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
  const int r = lane & 15, grp = lane >> 4;
  const int K = (int)a.K, steps = (K + kStep - 1) / kStep, tail = K - (steps - 1) * kStep;
  const int mine = steps > wave ? (steps - wave - 1) / WAVES + 1 : 0;
  const uint32_t ring = lds_at(lds) + wave * SLOTS * SLOT;
  uint32_t at[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) at[s] = ring + r * kStep + 16u * ((4 * s + grp) ^ swizzle(r));
  i32x4_t acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = i32x4_t{0, 0, 0, 0};
  auto operands = [&](uint32_t slot, u32x4_t (&w)[2][NT], u32x4_t (&x)[2][MT]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int n = 0; n < NT; ++n) w[s][n] = lds16(at[s] + slot + 16 * kStep * n);
#pragma unroll
      for (int m = 0; m < MT; ++m) x[s][m] = lds16(at[s] + slot + 16 * kStep * (NT + m));
    }
  };
  auto products = [&](const u32x4_t (&w)[2][NT], const u32x4_t (&x)[2][MT]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = mfma(w[s][n], x[s][m], acc[m][n]);
  };
  // piece i: rows 8 i .. of W, then of X; rows past the end repeat the last one
  auto row_of = [&](int i) {
    const int64_t r = (i < 2 * NT ? i : i - 2 * NT) * 8 + (lane >> 3);
    return min(r, (i < 2 * NT ? a.N - n0 : a.M - m0) - 1);
  };
  auto chunk_of = [&](int i) { return (lane & 7) ^ swizzle(8 * (i & 1) + (lane >> 3)); };
  const int8_t* const w_base = a.w + n0 * a.w_stride;
  const int8_t* const x_base = a.x + m0 * a.x_stride;
  if constexpr (DMA) {
    uint32_t off[P];
#pragma unroll
    for (int i = 0; i < P; ++i)
      off[i] = (uint32_t)(row_of(i) * (i < 2 * NT ? a.w_stride : a.x_stride)) + 16u * chunk_of(i);
    auto issue = [&](int i, uint32_t slot) {
      const int k = min((wave + i * WAVES) * kStep, K - kStep);
#pragma unroll
      for (int j = 0; j < P; ++j)
        dma(ring + slot + 1024 * j, (j < 2 * NT ? w_base : x_base) + k, off[j]);
    };
#pragma unroll
    for (int i = 0; i < RING; ++i)
      if (i < mine) issue(i, i * SLOT);
    uint32_t slot = 0;
    for (int i = 0; i < mine; ++i) {
      const int later = min(RING - 1, mine - 1 - i);   // steps still on their way
      if (later == 3) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(3 * P) : "memory");
      else if (later == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * P) : "memory");
      else if (later == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(P) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      u32x4_t w[2][NT], x[2][MT];
      operands(slot, w, x);
      if (wave + i * WAVES == steps - 1 && tail < kStep) {  // (K's last 128 bytes)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const bool in = 64 * s + 16 * grp >= kStep - tail;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int d = 0; d < 4; ++d) w[s][n][d] = in ? w[s][n][d] : 0u;
        }
      }
      // (read before the slot is filled again)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (i + RING < mine) issue(i + RING, slot);
      products(w, x);
      slot = slot + SLOT == RING * SLOT ? 0 : slot + SLOT;
    }
  } else {
    const int8_t* row[P];
#pragma unroll
    for (int i = 0; i < P; ++i)
      row[i] = i < 2 * NT ? w_base + row_of(i) * a.w_stride : x_base + row_of(i) * a.x_stride;
    u32x4_t held[RING][P];
    auto load = [&](int i, u32x4_t (&h)[P]) __attribute__((always_inline)) {
      if (i >= mine) return;
      const int k0 = (wave + i * WAVES) * kStep;
      if (k0 + kStep <= K) {
#pragma unroll
        for (int j = 0; j < P; ++j) h[j] = load16(row[j] + k0 + 16 * chunk_of(j));
      } else {
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const int k = k0 + 16 * chunk_of(j), from = min(k, K - 16);
          h[j] = load16(row[j] + from);
          if (j < 2 * NT) h[j] = without_first(h[j], k - from);
        }
      }
    };
#pragma unroll
    for (int i = 0; i < RING; ++i) load(i, held[i]);
    for (int i0 = 0; i0 < mine; i0 += RING)
#pragma unroll
      for (int u = 0; u < RING; ++u) {
        if (i0 + u >= mine) break;
#pragma unroll
        for (int j = 0; j < P; ++j)
          *(__attribute__((address_space(3))) u32x4_t*)(uintptr_t)(ring + 1024 * j + 16 * lane) =
              held[u][j];
        load(i0 + u + RING, held[u]);
        // (a wave's LDS accesses take effect in their order)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        u32x4_t w[2][NT], x[2][MT];
        operands(0, w, x);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        products(w, x);
      }
  }
  i32x4_t* const sums = (i32x4_t*)lds;   // [WAVES][Q][64], once no ring is in use
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) sums[(wave * Q + m * NT + n) * 64 + lane] = acc[m][n];
  __syncthreads();
  for (int q = wave; q < Q; q += WAVES) {
    const int64_t m = m0 + 16 * (q / NT) + r, n = n0 + 16 * (q % NT) + 4 * grp;
    i32x4_t s = sums[q * 64 + lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) s += sums[(v * Q + q) * 64 + lane];
    put4(a, m, n, s);
  }
}

// A row of fewer than 16 values: one result a thread.  (Bound by the launch and the results.)
__global__ void __launch_bounds__(256) int8_short_rows_kernel(LinearArgs a) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < a.M * a.N;
       e += (int64_t)gridDim.x * 256) {
    const int64_t m = e / a.N, n = e - m * a.N;
    int32_t sum = 0;
    for (int k = 0; k < a.K; ++k)
      sum += (int32_t)a.x[m * a.x_stride + k] * a.w[n * a.w_stride + k];
    const float y = scaled(sum, a.sx[m], a.sw[n], a.bias ? widen(a.bias, n, a.dtype) : 0.f);
    if (a.dtype == MRSA_DTYPE_FP32) ((float*)a.out)[e] = y;
    else ((uint16_t*)a.out)[e] = (uint16_t)pack2(y, 0.f, a.dtype);
  }
}

// Rows of any stride and address to rows of `padded` bytes (a multiple of 128), zeros behind
// K >= 16: W's N rows, then X's M.  16 bytes a thread; blocks cover chunks (x) of rows (y).  Bound
// by its bytes: 16384 + 3584 rows of 18943, 757 MB read and written, about 130 us (5.8 TB/s).
__global__ void __launch_bounds__(256) int8_pad_kernel(LinearArgs a, int64_t padded, int8_t* to) {
  const int64_t k = 16 * ((int64_t)blockIdx.x * blockDim.x + threadIdx.x);
  if (k >= padded) return;
  for (int64_t r = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; r < a.N + a.M;
       r += (int64_t)gridDim.y * blockDim.y) {
    const int8_t* const from = r < a.N ? a.w + r * a.w_stride : a.x + (r - a.N) * a.x_stride;
    u32x4_t v = {0, 0, 0, 0};
    if (k + 16 <= a.K) {
      v = load16(from + k);
    } else if (k < a.K) {
      // the row's last 16 bytes, the ones before k moved out
      v = load16(from + a.K - 16);
      const int out = 16 - (int)(a.K - k), words = out >> 2, bits = 8 * (out & 3);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e == d + words) lo = v[e];
          if (e == d + words + 1) hi = v[e];
        }
        // (d ascends and reads only what is at or above it)
        v[d] = bits ? lo >> bits | hi << (32 - bits) : lo;
      }
    }
    *(u32x4_t*)(to + r * padded + k) = v;
  }
}

// How a product is cut: by its sizes and alignment alone.  A step of a tile costs about the same
// for few rows as for many, so small tiles finish few rows first and large ones many; `parts` of K
// fill the CUs where tiles do not, for a second kernel's time.  The estimate below is fitted to
// measured times (us; 64 to 16384 rows, 64 to 37888 columns, 1008 to 18944 values).
//   512 rows, 3584 x 3584: 64 x 64 16.3, 64 x 128 14.7, 128 x 128 18.1, 256 x 256 42
//   256 rows, 3584 columns of 18944 values: 64 x 64 55 (two parts 48), 128 x 128 83 (four 32)
//   1003 rows of the same: 64 x 64 138, 128 x 128 87, 256 x 256 230 (four 86)
//   128 rows, 37888 x 3584: 128 x 256 34, 128 x 128 40, 256 x 256 50
//   4096 rows, 8192 x 8192: 256 x 256 223, 128 x 256 258, 128 x 128 280
typedef Tile<64, 64, 2, 1, 4, 4> Tile64;
typedef Tile<64, 128, 2, 2, 3, 3> Tile64x128;
typedef Tile<128, 128, 4, 2, 4, 4> TileDeep;     // a workgroup a CU
typedef Tile<128, 128, 4, 2, 2, 2> Tile128;      // two
typedef Tile<128, 256, 2, 4, 3, 3> Tile128x256;
typedef Tile<256, 256, 2, 4, 3, 2> Tile256;
struct Shape {
  int tm, tn, room;        // workgroups that the CUs hold
  float one, two, fixed;   // us: a step of a workgroup alone on its CU, of two, the rest
  float any_rows;          // a step's time of rows at any address over that of aligned ones (0: -)
};
constexpr Shape kShapes[] = {
    {64, 64, 512, 0.335f, 0.45f, 5.f, 1.9f},  {64, 128, 512, 0.40f, 0.70f, 5.f, 0.f},
    {128, 128, 256, 0.52f, 0.52f, 5.f, 0.f},  {128, 128, 512, 0.83f, 1.0f, 5.f, 1.6f},
    {128, 256, 256, 0.82f, 0.82f, 6.f, 0.f},  {256, 256, 256, 1.42f, 1.42f, 8.f, 1.6f},
};
struct Plan {
  enum { kShort, kFew, kTiles } kind;
  int shape;
  bool dma;
  int64_t tiles_m, tiles_n, parts, bytes, cols;
  int64_t padded;   // bytes of the padded rows that the tiles are cut from, at the workspace's end
};

// The best cut of tiles that beats `best` us, with `more` us for all that comes before them.
void best_tiles(int64_t M, int64_t N, int64_t K, bool aligned, float more, float& best, Plan& p) {
  const int64_t steps = (K + kStep - 1) / kStep;
  for (int i = 0; i < (int)(sizeof(kShapes) / sizeof(kShapes[0])); ++i) {
    const Shape& s = kShapes[i];
    if (!aligned && s.any_rows == 0.f) continue;
    const int64_t tm = (M + s.tm - 1) / s.tm, tn = (N + s.tn - 1) / s.tn;
    for (const int parts : {1, 2, 3, 4, 6, 8}) {
      if (parts > steps) break;
      const int64_t items = tm * tn * parts;
      if (parts > 1 && items > s.room) break;  // (and so the workspace stays small)
      const float rounds = items <= 4 * s.room ? (float)((items + s.room - 1) / s.room)
                                               : (float)items / (float)s.room + 0.5f;
      const float step = (items <= 256 ? s.one : s.two) * (aligned ? 1.f : s.any_rows);
      const int64_t bytes = parts > 1 ? items * s.tm * s.tn * 4 : 0;
      const float time = more +
                         rounds * (s.fixed + step * (float)((steps + parts - 1) / parts)) +
                         (parts > 1 ? 6.f + 0.27e-6f * (float)bytes : 0.f);
      if (time < best) {
        best = time;
        p = {Plan::kTiles, i, aligned, tm, tn, parts, bytes, 0, 0};
      }
    }
  }
}

// Rows by 64, through the kernel of few rows: as long as its workgroups are one round or two, since
// a wave takes a quarter of K's steps and no barriers (us, its 16 and 32 columns, and tiles: 512
// rows, 1008 x 1008 4.7, 5.5 and 6.8; 64 x 3584 5.5, 6.8 and 9.5; 128 rows, 3584 x 3584 9.4, 7.6
// and 13.7, of 3583 values 16, 12 and 17; 192 rows 12.5, 13.1 and 13.8; 256 rows 15, 13 and 14; 128
// rows, 4608 x 3584 12.6, 13.2 and 13.7, 8192 x 4096 21, 18 and 16).  The estimate: rounds; or the
// bytes that all workgroups fetch, W's again for each 64 rows and the rows' for each 16 or 32
// columns; or those of them that come from beyond the L2s, each of which sees all workgroups.
void best_few(int64_t M, int64_t N, int64_t K, bool aligned, float& best, Plan& p) {
  const int64_t tm = (M + 63) / 64, steps = (K + 4 * kStep - 1) / (4 * kStep);
  if (tm > 65535) return;
  for (const int cols : {16, 32}) {
    const int64_t tn = (N + cols - 1) / cols, items = tm * tn;
    float rounds, step, rate;   // rate: bytes a us
    if (cols == 16) {
      rounds = std::max(1.f, (float)items / 512.f);
      step = aligned ? (items <= 256 ? 0.57f : 0.97f) : (items <= 256 ? 1.0f : 2.05f);
      rate = aligned ? 16.5e6f : 9.4e6f;
    } else {
      rounds = (float)((items + 255) / 256);
      step = aligned ? 0.72f : 1.3f;
      rate = aligned ? 12e6f : 7.5e6f;
    }
    const float bytes = (float)tm * (float)N * (float)K * (1.f + 64.f / (float)cols);
    const float far = (float)K * ((float)N * (float)std::min<int64_t>(tm, 8) +
                                  (float)M * (float)std::min<int64_t>(tn, 8));
    const float time = 1.2f + std::max(rounds * (2.f + step * (float)steps),
                                       2.f + std::max(bytes / rate, far / 5.5e6f));
    if (time < best) {
      best = time;
      p = {Plan::kFew, 0, aligned, tm, tn, 1, 0, cols, 0};
    }
  }
}

Plan plan_of(int64_t M, int64_t N, int64_t K, bool aligned) {
  Plan p = {Plan::kTiles, 0, aligned, 1, 1, 1, 0, 0, 0};
  if (K < 16) {
    p.kind = Plan::kShort;
    return p;
  }
  if (M <= 32) {
    // The weights' bytes count.  Columns of a workgroup: 32 while that leaves half the CUs a
    // workgroup, else 16 (us, 16 and 32: 32 rows of 3584 values, 3584 columns 5.0 and 5.3, 4608 6.8
    // and 5.6, 37888 39 and 31; 16 rows of 4096, 4096 columns 6.9 and 5.9).
    p.kind = Plan::kFew;
    p.cols = N >= 32 * 128 ? 32 : 16;
    p.tiles_n = (N + p.cols - 1) / p.cols;
    return p;
  }
  float best = 1e30f;
  best_few(M, N, K, aligned, best, p);
  best_tiles(M, N, K, aligned, 0.f, best, p);
  if (K % 16 != 0) {
    // Rows that no stride aligns: padded copies of them first where the tiles gain more than the
    // copies' bytes cost (us, through registers and with copies: 512 x 3584 of 3583 values 27.9 and
    // 26.3, 2000 x 2000 of 7999 70 and 51, 8192 x 4096 of 4095 161 and 139, 16384 x 3584 of 18943
    // 1451 and 1095).
    const int64_t padded = (K + kStep - 1) / kStep * kStep;
    const float bytes = (float)(M + N) * (float)padded;
    const float before = best;
    best_tiles(M, N, padded, true, 3.f + bytes * 0.33e-6f, best, p);
    if (best < before) {
      p.padded = padded;
      p.bytes += (M + N) * padded;
    }
  }
  return p;
}
bool aligned_rows(const void* p, int64_t stride, int64_t rows) {
  return (uintptr_t)p % 16 == 0 && (rows == 1 || (stride % 16 == 0 && stride < (1 << 22)));
}

template <class T, bool ANY>
void launch_tiles(const LinearArgs& a, bool dma, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.tiles_m * a.tiles_n * a.parts)), block(T::THREADS);
  if (dma) {
    hipLaunchKernelGGL((int8_tile_kernel<T, true>), grid, block, 0, stream, a);
  } else if constexpr (ANY) {
    hipLaunchKernelGGL((int8_tile_kernel<T, false>), grid, block, 0, stream, a);
  }
  if (a.parts > 1)
    hipLaunchKernelGGL((int8_join_kernel<T>),
                       dim3((unsigned)(a.tiles_m * a.tiles_n * (T::MT * T::NT / 2))), block, 0,
                       stream, a);
}

template <bool DMA>
void launch_few(const LinearArgs& a, const Plan& p, hipStream_t stream) {
  const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
  void (*kern)(LinearArgs);
  if (p.cols == 16)
    kern = mt == 1   ? int8_stream_kernel<1, 1, 4, 4, DMA>
           : mt == 2 ? int8_stream_kernel<2, 1, 4, 3, DMA>
                     : int8_stream_kernel<4, 1, 4, 2, DMA>;
  else
    kern = mt == 1   ? int8_stream_kernel<1, 2, 4, 2, DMA>
           : mt == 2 ? int8_stream_kernel<2, 2, 4, 2, DMA>
                     : int8_stream_kernel<4, 2, 4, 2, DMA>;
  hipLaunchKernelGGL(kern, dim3((unsigned)p.tiles_n, (unsigned)p.tiles_m), dim3(256), 0, stream, a);
}

}  // namespace

extern "C" int64_t mrsa_int8_linear_workspace_bytes(int64_t rows, int64_t out_dim, int64_t dim) {
  if (rows < 0 || out_dim < 0 || dim < 0 || rows >= (int64_t)1 << 31 ||
      out_dim >= (int64_t)1 << 31 || dim > 131071)
    return -1;
  const int64_t bytes = plan_of(rows, out_dim, dim, false).bytes;
  return dim % 16 != 0 ? bytes : std::max(bytes, plan_of(rows, out_dim, dim, true).bytes);
}

extern "C" int mrsa_int8_linear_fwd(const int8_t* x, int64_t x_row_stride, const float* x_scales,
                                    const int8_t* weight, int64_t weight_row_stride,
                                    const float* weight_scales, const void* bias, int64_t rows,
                                    int64_t out_dim, int64_t dim, int32_t dtype, void* workspace,
                                    int64_t workspace_bytes, void* out, void* stream) {
  if (rows < 0 || out_dim < 0 || dim < 0 || x_row_stride < 0 || weight_row_stride < 0)
    return MRSA_ERR_INVALID_ARGUMENT;
  if (dtype != MRSA_DTYPE_BF16 && dtype != MRSA_DTYPE_FP16 && dtype != MRSA_DTYPE_FP32)
    return MRSA_ERR_UNSUPPORTED;
  if (dim > 131071 || rows >= (int64_t)1 << 31 || out_dim >= (int64_t)1 << 31 ||
      x_row_stride >= (int64_t)1 << 31 || weight_row_stride >= (int64_t)1 << 31)
    return MRSA_ERR_UNSUPPORTED;
  if (rows == 0 || out_dim == 0) return MRSA_OK;
  const int size = dtype == MRSA_DTYPE_FP32 ? 4 : 2;
  if (!x_scales || !weight_scales || !out || (dim > 0 && (!x || !weight)))
    return MRSA_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)x_scales | (uintptr_t)weight_scales) % 4 != 0 ||
      ((uintptr_t)bias | (uintptr_t)out) % size != 0)
    return MRSA_ERR_INVALID_ARGUMENT;
  const bool aligned = dim % 16 == 0 && dim >= kStep && aligned_rows(x, x_row_stride, rows) &&
                       aligned_rows(weight, weight_row_stride, out_dim);
  const Plan p = plan_of(rows, out_dim, dim, aligned);
  const int64_t groups = p.tiles_m * p.tiles_n * p.parts;
  if (groups >= (int64_t)1 << 23) return MRSA_ERR_UNSUPPORTED;
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || (uintptr_t)workspace % 16 != 0))
    return MRSA_ERR_INVALID_ARGUMENT;
  LinearArgs a = {x, weight, x_scales, weight_scales, bias, out, (int32_t*)workspace, rows,
                        out_dim, dim, x_row_stride, weight_row_stride, dtype, (int32_t)p.parts,
                        (int32_t)p.tiles_m, (int32_t)p.tiles_n};
  const hipStream_t st = (hipStream_t)stream;
  if (p.padded > 0) {
    int8_t* const to = (int8_t*)workspace + (p.bytes - (rows + out_dim) * p.padded);
    const int64_t chunks = p.padded / 16, all = rows + out_dim;
    unsigned tx = 8;
    while (tx < 64 && tx < chunks) tx *= 2;
    const dim3 block(tx, 256 / tx);
    const int64_t by = std::min<int64_t>((all + block.y - 1) / block.y, 16384);
    hipLaunchKernelGGL(int8_pad_kernel, dim3((unsigned)((chunks + tx - 1) / tx), (unsigned)by),
                       block, 0, st, a, p.padded, to);
    a.w = to;
    a.x = to + out_dim * p.padded;
    a.K = a.x_stride = a.w_stride = p.padded;
  }
  switch (p.kind) {
    case Plan::kShort: {
      const int64_t blocks = std::min<int64_t>((rows * out_dim + 255) / 256, 1 << 20);
      hipLaunchKernelGGL(int8_short_rows_kernel, dim3((unsigned)blocks), dim3(256), 0, st, a);
      break;
    }
    case Plan::kFew: {
      if (p.dma) launch_few<true>(a, p, st);
      else launch_few<false>(a, p, st);
      break;
    }
    case Plan::kTiles:
      switch (p.shape) {
        case 0: launch_tiles<Tile64, true>(a, p.dma, st); break;
        case 1: launch_tiles<Tile64x128, false>(a, p.dma, st); break;
        case 2: launch_tiles<TileDeep, false>(a, p.dma, st); break;
        case 3: launch_tiles<Tile128, true>(a, p.dma, st); break;
        case 4: launch_tiles<Tile128x256, false>(a, p.dma, st); break;
        default: launch_tiles<Tile256, true>(a, p.dma, st);
      }
      break;
  }
  return mrsa_launch_status();
}
