// Attention of the newest rows of several sequences against a paged K/V cache,
// split over the cache's length and joined.
//
// Sequence b holds n = cache_lens[b] rows; its query row i sits at position
// p = query_starts[b] + i (by default the query rows are the last ones).  A
// row with p in [0, n) sees the keys j of [0, n) with j <= p if causal,
// |j - p| <= window if windowed, that lie in a mapped page (an entry of the
// page table outside [0, num_pages) holds no keys); other rows are padding:
//   s_j = scale q . k_j,  lse = log sum_j exp s_j,  out = sum_j exp(s_j - lse) v_j,
// and out = 0, lse = -inf for a row that sees none.
//
// The G query heads of a KV head and the q_len rows are matrix columns
// (column m: row m / G, head m % G).  Tiles of keys are passed once, with a running
// maximum and sum per column:
//   S^T = K . Q^T    K rows as operand A
//   O^T += V^T . P^T P^T is S^T's own register layout (operand B); V comes
//                    transposed from LDS (gfx950's transposing reads).
// Products of 16-bit inputs are exact, sums fp32; P is rounded to the inputs'
// type as a matrix operand (the sum uses the unrounded values), which is half
// a step of that type per term.  The maximum moves only when scores have passed it
// by some powers of two, so that the accumulators are rarely rescaled.
// fp16 reaches down to 2^-24 only, and many weights below that can be much of a row's sum: they
// are taken times 2^lift (the running maximum is held that much lower; sums and outputs have
// the same factor), which the room up to the moving maximum and fp16's largest value leave.
// What a weight then loses is below 2^-25 / 2^lift of the largest: 20000 keys of 2^-25.2 gave
// 0 of the output's 5.0e-4 before.
//
// Up to 16 columns (a token's heads) the work is the cache's bytes: `paged_attn_kernel`
// streams them.  With more columns every key is multiplied often enough to be
// brought to LDS once for all: `paged_block_kernel`.  8 sequences of 8191 keys of 4 KV
// heads: 14 columns 30 us by the former, 21 columns 32 by the latter, 48 by two tiles
// of the former.  `parts` cuts the keys of a sequence into pieces for workgroups of
// their own, where there are few; fp32 partial results go through a workspace to
// `paged_join_kernel`.
#include "chunk_tile.h"
#include "mrsa_device.h"

using namespace mrsa;

namespace {

constexpr int kWaves = 4;                  // of the streaming kernel
constexpr int kTile = 32;                  // keys of a wave's tile
constexpr int kStep = kWaves * kTile;      // keys of a workgroup's round
// LDS of a streaming workgroup: more than it needs, so that two are on a CU and not three: 64
// sequences of 1024 to 8192 keys in three pieces then take 128 us, 155 with three on a CU, and
// the other lengths and numbers of pieces differ by less.
constexpr int kStreamLds = 56 * 1024;
constexpr int kMaxParts = 1024;
constexpr int kFar = 1 << 29;              // bound of positions and windows: their sums fit 32 bits
constexpr float kSlack = 8.f;              // base-2 growth before the maximum moves
constexpr float kMostSum = 1024.f;         // sum of sixteen weights before it moves (block kernel)

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

struct Bf16 {
  static __device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return mfma_bf16_16x16x32(a, b, c);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return pack_bf16x2(lo, hi);
  }
  static __device__ __forceinline__ float value(uint32_t bits) { return bf16_to_f32(bits); }
  static constexpr uint32_t kExp = 0x7f80u;
  static constexpr float kStreamLift = 0.f, kBlockLift = 0.f;   // (exponents as fp32's)
};
struct Fp16 {
  static __device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    f32x2_t v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
  }
  static __device__ __forceinline__ float value(uint32_t bits) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  }
  static constexpr uint32_t kExp = 0x7c00u;
  // weights below 2^(kSlack + 7) and kMostSum 2^5: 2^15
  static constexpr float kStreamLift = 7.f, kBlockLift = 5.f;
};

struct PagedArgs {
  const uint16_t* q;
  int64_t q_sb, q_sl, q_sh;
  const uint16_t* k;
  int64_t k_sp, k_sr, k_sh;   // page, row, head strides
  const uint16_t* v;
  int64_t v_sp, v_sr, v_sh;
  const int32_t* table;
  int64_t table_stride;
  int table_width, page_shift, num_pages;
  const int32_t* lens;
  const int32_t* starts;      // optional
  int max_len;
  int B, Lq, Hq, Hkv, G, M;   // M = Lq G columns
  int causal, window;         // window < 0: none
  float scale_log2;
  int parts, part_keys, col_tiles, tile_cols;
  uint16_t* out;
  float* lse;
  float* part_out;            // parts > 1: [B, Hkv, M, parts, D]
  float* part_ml;             // parts > 1: [B, Hkv, M, parts, 2]
};

// Page table and lengths are read through the constant address space, that is by
// scalar loads (nothing writes them while the kernel runs): a vector load's
// result would be waited for behind every K and V load in flight.
typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
__device__ __forceinline__ scalar_ints scalars(const int32_t* p) {
  return (scalar_ints)(uintptr_t)p;
}
// The kernel's arguments, to be read again: what only a kernel's end or a rare path needs would
// otherwise hold scalar registers through its loop.
typedef const __attribute__((address_space(4))) PagedArgs* args_again_t;
__device__ __forceinline__ args_again_t args_again() {
  args_again_t p = (args_again_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}
// The page of sixteen keys from `key` on (wave-uniform); -1 past the table.
__device__ __forceinline__ int page_at(const PagedArgs& a, scalar_ints table, int key) {
  const int e = key >> a.page_shift;
  const int page = table[min(e, a.table_width - 1)];
  return e < a.table_width ? page : -1;
}

// Rows in use of sequence b.
__device__ __forceinline__ int length_of(const PagedArgs& a, int b) {
  const int n = min(scalars(a.lens)[b], a.max_len);
  const int64_t room = (int64_t)a.table_width << a.page_shift;
  return max(0, (int)min((int64_t)n, room));
}
// Position of query row 0 of sequence b.
__device__ __forceinline__ int start_of(const PagedArgs& a, int b, int n) {
  return a.starts ? max(-kFar, min(kFar, scalars(a.starts)[b])) : n - a.Lq;
}
// Keys [lo, hi) that the row at position p of [0, n) may see, both rising with p.
__device__ __forceinline__ void seen_by(const PagedArgs& a, int n, int p, int& lo, int& hi) {
  lo = a.window >= 0 ? max(0, min(n, p - a.window)) : 0;
  hi = n;
  if (a.causal) hi = min(hi, p + 1);
  if (a.window >= 0) hi = min(hi, p + a.window + 1);
  hi = max(0, hi);
}
// Keys of a column tile: [start, end) that some column sees (start a multiple
// of the tile), [inner_lo, inner_hi) that all see.
struct Range {
  int start, end, inner_lo, inner_hi, lo;
};
__device__ __forceinline__ Range tile_range(const PagedArgs& a, int n, int p0, int first_col,
                                            int cols) {
  // first and last position of the tile's rows that are not padding
  const int pa = max(0, p0 + first_col / a.G);
  const int pz = min(n - 1, p0 + min(a.M - 1, first_col + cols - 1) / a.G);
  Range r = {0, 0, 0, 0, 0};
  if (pz < pa) return r;
  seen_by(a, n, pa, r.lo, r.inner_hi);
  seen_by(a, n, pz, r.inner_lo, r.end);
  r.start = r.lo & ~(kTile - 1);
  return r;
}

// Whether some column, not every one, sees a key of [base, base + keys).
__device__ __forceinline__ bool is_uneven(const Range& r, int base, int keys) {
  return max(base, r.lo) < r.inner_lo || min(base + keys, r.end) > r.inner_hi;
}

// Swizzle of V's LDS rows in 16-byte units: the transposing read's rows of one
// lane group meet different banks.
template <int D>
__device__ __forceinline__ int swizzle(int r) {
  return D == 128 ? 2 * (r & 7) + ((r >> 3) & 1) : 2 * ((r >> 1) & 3) + ((r >> 3) & 1);
}

// Up to 16 columns.  A workgroup's four waves take tiles of 32 keys in turn: K rows straight
// from HBM to registers, V rows through the wave's own piece of LDS, a tile's loads
// in flight while the one before is worked on.  Bound by HBM: 131072 keys of 4 KV heads,
// 256 MB, in 50.4 us, 5.3 TB/s, a large copy's rate; 64 sequences of 1024 to 8192 keys, 584 MB, in
// 122 us, 5.0 TB/s; 1000 keys in 5.8 us, the launch and three dependent reads.  (Without the
// bound on registers the compiler moves the accumulators between register files every
// tile: 0.8 us more for a token.)
template <class T, int D>
__global__ void __launch_bounds__(64 * kWaves, 2) paged_attn_kernel(PagedArgs a) {
  constexpr int KS = D / 32;             // reduction steps of S
  constexpr int DT = D / 16;             // output tiles
  constexpr int UNITS = D / 8;           // 16-byte units of a row
  constexpr int VROWS = 64 / UNITS;      // rows of one V load
  constexpr int VL = kTile / VROWS;      // V loads per lane
  constexpr int ROWB = 2 * D;            // bytes of a row
  constexpr int OPAD = D + 4;
  extern __shared__ __align__(256) unsigned char smem[];
  __shared__ float red_m[kWaves][16], red_l[kWaves][16];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  uint32_t id = blockIdx.x;  // (the grid is below 2^31)
  // KV heads next to each other (a row's heads are neighbours in memory), parts last: of
  // sequences of different lengths the short pieces at their ends then come last.
  const int h = id % (uint32_t)a.Hkv;
  id /= (uint32_t)a.Hkv;
  const int ct = id % (uint32_t)a.col_tiles;
  id /= (uint32_t)a.col_tiles;
  const int b = id % (uint32_t)a.B;
  const int part = id / (uint32_t)a.B;

  const int n = length_of(a, b), p0 = start_of(a, b, n);
  const Range r = tile_range(a, n, p0, ct * 16, 16);
  const int first = r.start + part * a.part_keys;
  const int last = min(r.end, first + a.part_keys);
  if (part > 0 && first >= r.end) return;   // (part 0 also writes the empty rows)

  // ---- this lane's column
  const int m = ct * 16 + col;
  const bool cok = m < a.M;
  const int qi = cok ? m / a.G : 0, qg = cok ? m - qi * a.G : 0;
  const int pos = p0 + qi;
  const bool padding = !cok || pos < 0 || pos >= n;
  int lo = 0, hi = 0;
  if (!padding) seen_by(a, n, pos, lo, hi);
  u32x4_t Q[KS];
  {
    const uint16_t* qp = a.q + b * a.q_sb + qi * a.q_sl + (h * a.G + qg) * a.q_sh + 8 * grp;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Q[s] = u32x4_t{0, 0, 0, 0};
      if (cok) Q[s] = *reinterpret_cast<const u32x4_t*>(qp + 32 * s);
    }
  }
  f32x4_t O[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) O[t] = zero4();
  float mx = neg_inf(), sum = 0.f;

  const scalar_ints table = scalars(a.table + b * a.table_stride);
  const int page_mask = (1 << a.page_shift) - 1;
  const uint16_t* kb = a.k + h * a.k_sh + col * a.k_sr + 8 * grp;
  const int vrow = lane / UNITS, vunit = lane % UNITS;
  const uint16_t* vb = a.v + h * a.v_sh + vrow * a.v_sr + 8 * vunit;
  unsigned char* vl = smem + wave * kTile * ROWB;
  const uint32_t vbase = lds_addr(vl);
  // transposing reads: row 4 grp + (col >> 2), piece col & 3 of its 32 bytes
  const int tr = 4 * grp + (col >> 2);
  const uint32_t tr0 =
      vbase + tr * ROWB + ((((col & 3) >> 1) ^ swizzle<D>(tr)) << 4) + (col & 1) * 8;

  // Every load is issued a tile ahead: V's as soon as the registers have gone
  // to LDS, K's after the products, page indices one tile before those.
  u32x4_t K[2][KS], V[VL];
  int pages[2], next_pages[2];  // of the tile's sixteens of keys
  auto page_of = [&](int key) { return page_at(a, table, key); };
  auto is_live = [&](int page) { return page >= 0 && page < a.num_pages; };
  auto safe = [&](int page) { return is_live(page) ? page : 0; };  // a page that exists
  auto load_k = [&](int base, const int (&pg)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t* kp = kb + safe(pg[t]) * a.k_sp + ((base + 16 * t) & page_mask) * a.k_sr;
#pragma unroll
      for (int s = 0; s < KS; ++s) K[t][s] = *reinterpret_cast<const u32x4_t*>(kp + 32 * s);
    }
  };
  auto load_v = [&](int base, const int (&pg)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint16_t* vp = vb + safe(pg[t]) * a.v_sp + ((base + 16 * t) & page_mask) * a.v_sr;
#pragma unroll
      for (int i = 0; i < VL / 2; ++i)
        V[t * (VL / 2) + i] = *reinterpret_cast<const u32x4_t*>(vp + i * VROWS * a.v_sr);
    }
  };
  const int begin = first + wave * kTile;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    pages[t] = begin < last ? page_of(begin + 16 * t) : -1;
    next_pages[t] = begin + kStep < last ? page_of(begin + kStep + 16 * t) : -1;
  }
  if (begin < last) {
    load_v(begin, pages);
    load_k(begin, pages);
  }
  for (int base = begin; base < last; base += kStep) {
    const bool live[2] = {is_live(pages[0]), is_live(pages[1])};
    const bool more = base + kStep < last;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      pages[t] = next_pages[t];
      next_pages[t] = base + 2 * kStep < last ? page_of(base + 2 * kStep + 16 * t) : -1;
    }
    const bool whole = live[0] && live[1];
    const bool edge = !whole || base < r.lo || base + kTile > r.end;           // V rows nobody sees
    const bool mixed = !whole || base < r.inner_lo || base + kTile > r.inner_hi;  // masked scores
    uint64_t dirty = 0;
    if (edge) {  // rows nobody sees become zeros
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int key = base + i * VROWS + vrow;
        const bool there = live[i / (VL / 2)] && key >= r.lo && key < r.end;
        if (!there) V[i] = u32x4_t{0, 0, 0, 0};
      }
    }
    if (is_uneven(r, base, kTile)) {
      // Keys that some columns see and others do not: a non-finite value
      // must not reach the others as 0 x inf, so it is taken out here and its
      // terms are added one by one below.
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t w = V[i][e];
          const bool b0 = (w & T::kExp) == T::kExp, b1 = ((w >> 16) & T::kExp) == T::kExp;
          odd |= b0 || b1;
          if (b0) w &= 0xffff0000u;
          if (b1) w &= 0x0000ffffu;
          V[i][e] = w;
        }
        dirty |= __builtin_amdgcn_ballot_w64(odd);
      }
    }
    // ---- V to LDS
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int rr = i * VROWS + vrow;
      *reinterpret_cast<u32x4_t*>(vl + rr * ROWB + ((vunit ^ swizzle<D>(rr)) << 4)) = V[i];
    }
    if (more) load_v(base + kStep, pages);
    // ---- scores
    f32x4_t S[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      S[t] = zero4();
#pragma unroll
      for (int s = 0; s < KS; ++s) S[t] = T::mfma(K[t][s], Q[s], S[t]);
    }
    if (more) load_k(base + kStep, pages);
    uint32_t seen = 0xffu;
    if (mixed) {
      seen = 0;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = base + 16 * t + 4 * grp + e;
          const bool ok = live[t] && key >= lo && key < hi;
          if (ok) seen |= 1u << (4 * t + e);
          S[t][e] = ok ? S[t][e] : neg_inf();
        }
    }
    float top = S[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, S[i >> 2][i & 3]);
    top = across4_max(top) * a.scale_log2;   // (-inf stays: the scale is positive)
    if (__builtin_amdgcn_ballot_w64(top > mx + (kSlack + T::kStreamLift)) != 0) {
      const float to = __builtin_fmaxf(mx, top - T::kStreamLift);
      const float f = to == neg_inf() ? 1.f : exp2_hw(mx - to);
      mx = to;
      sum *= f;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[t][e] *= f;
    }
    const float off = mx == neg_inf() ? 0.f : mx;
    float P[8];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        P[4 * t + e] = exp2_hw(__builtin_fmaf(S[t][e], a.scale_log2, -off));
        sum += P[4 * t + e];
      }
    const u32x4_t Pb = {T::pack(P[0], P[1]), T::pack(P[2], P[3]), T::pack(P[4], P[5]),
                        T::pack(P[6], P[7])};
    // ---- V^T . P^T
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const uint32_t at = tr0 ^ (t << 5);
      const u32x2_t x = read_transposed(at), y = read_transposed(at + 16 * ROWB);
      O[t] = T::mfma(u32x4_t{x[0], x[1], y[0], y[1]}, Pb, O[t]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (dirty) {
      for (int kk = 0; kk < kTile; ++kk) {
        const int key = base + kk;
        if (!live[kk >> 4] || key < r.lo || key >= r.end) continue;
        const int from = 16 * ((kk & 15) >> 2) + col;
        const int slot = 4 * (kk >> 4) + (kk & 3);
        const bool ok = (__shfl(seen, from, 64) >> slot) & 1;
        const uint16_t* vp =
            a.v + h * a.v_sh + page_of(key) * a.v_sp + (key & page_mask) * a.v_sr;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t w = vp[16 * t + 4 * grp + e];
            // (p > 0: its size is no matter)
            if (ok && (w & T::kExp) == T::kExp) O[t][e] += T::value(w);
          }
      }
    }
  }

  // ---- join the four waves
  if (padding) {  // (its scores were not masked in tiles that every row sees)
    mx = neg_inf();
    sum = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t) O[t] = zero4();
  }
  sum = across4_sum(sum);
  if (grp == 0) {
    red_m[wave][col] = mx;
    red_l[wave][col] = sum;
  }
  __syncthreads();
  float M = neg_inf(), total = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) M = __builtin_fmaxf(M, red_m[w][col]);
  const float f = M == neg_inf() ? 1.f : exp2_hw(mx - M);
  float* ol = reinterpret_cast<float*>(smem) + wave * 16 * OPAD + col * OPAD;
#pragma unroll
  for (int t = 0; t < DT; ++t)
    *reinterpret_cast<f32x4_t*>(ol + 16 * t + 4 * grp) = O[t] * f;
  __syncthreads();
  // thread: column tid / TPC, DPT dims
  constexpr int TPC = 64 * kWaves / 16, DPT = D / TPC;
  const int c2 = tid / TPC, d2 = (tid % TPC) * DPT;
  const int m2 = ct * 16 + c2;
  if (m2 >= a.M) return;
  M = neg_inf();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) M = __builtin_fmaxf(M, red_m[w][c2]);
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    total += red_l[w][c2] * (M == neg_inf() ? 1.f : exp2_hw(red_m[w][c2] - M));
  float acc[DPT];
#pragma unroll
  for (int d = 0; d < DPT; ++d) acc[d] = 0.f;
  for (int w = 0; w < kWaves; ++w)
#pragma unroll
    for (int d = 0; d < DPT; ++d)
      acc[d] += reinterpret_cast<float*>(smem)[w * 16 * OPAD + c2 * OPAD + d2 + d];
  if (a.parts > 1) {
    const int64_t at = (((int64_t)b * a.Hkv + h) * a.M + m2) * a.parts + part;
#pragma unroll
    for (int d = 0; d < DPT; ++d) a.part_out[at * D + d2 + d] = acc[d];
    if (d2 == 0) {
      a.part_ml[2 * at] = M;
      a.part_ml[2 * at + 1] = total;
    }
    return;
  }
  const int i2 = m2 / a.G;
  const int64_t row = ((int64_t)b * a.Lq + i2) * a.Hq + h * a.G + (m2 - i2 * a.G);
  const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
  for (int d = 0; d < DPT; d += 2)
    *reinterpret_cast<uint32_t*>(a.out + row * D + d2 + d) =
        total == 0.f ? 0u : T::pack(acc[d] * inv, acc[d + 1] * inv);
  if (d2 == 0) a.lse[row] = total == 0.f ? neg_inf() : kLn2 * (M + log2_hw(total));
}

// Many columns: a workgroup of up to eight waves, 32 columns each, over tiles of
// 64 keys that all its waves read from LDS.  K and V rows come by global->LDS
// DMA into a ring, a tile ahead, one barrier per tile; K is read along the row
// (operand A of S^T), V by transposing reads (operand A of O^T).
//
// Bound by what lies between its units: a wave's tile is 64 matrix instructions and about 130
// vector ones (32 exponentials, their arguments, the sums, the packing), two waves share a
// SIMD, and in a long loop (8192 rows of 8192 keys) the matrix cores and the vector unit are at
// work for 45 and 43% of the cycles, with waves waiting a fifth of theirs at the tile's barrier and
// for operands; with few rows and all CUs at work HBM comes near, too.  So the two go half a
// tile apart (the softmax of one runs beside the products of the other), tiles that every
// column sees whole have a loop of their own without masks, with the ring's slots as
// constants, the maximum is not taken per tile, and the next rows' addresses are computed
// before the barrier.  28 heads in 4 groups, 32 rows, 65503 keys (30
// GFLOP, 134 MB; 64 pieces): 43.4 us, 690 TFLOP/s; of them 5 until the first rows are there, 28
// for sixteen tiles (1.45 us a tile with few workgroups, more with 256, which stream 3.7 TB/s)
// and 8 for the partial results' way out.  Without the one after the other: addresses
// behind the barrier 45.2, slots as variables 47.8, a maximum per tile 49.7, masks and waves
// in step 54.
constexpr int kBlockKeys = 64;
constexpr int kBlockCols = 32;             // of a wave
constexpr int kBlockWaves = 8;

// A piece by DMA: N instructions, each 1 KB of LDS from `to` on, lane l's 16 bytes from
// base + at[i].  As asm, since after the builtin the compiler waits for all DMA in flight before
// the next LDS read; here the loop's own waits order them.  base and to are
// wave-uniform; the first s_nop covers a scalar operand that a vector instruction
// has just written (5 wait states), the others m0.
template <int N>
__device__ __forceinline__ void dma_piece(uint32_t to, const uint8_t* base,
                                          const uint32_t (&at)[N]) {
  static_assert(N == 2 || N == 4);
  if constexpr (N == 4)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %2, %1\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %1\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %1\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %1" ::"s"(to),
        "s"(base), "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[N - 1])
        : "memory", "m0", "scc");
  else
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %2, %1\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %1" ::"s"(to),
        "s"(base), "v"(at[0]), "v"(at[1])
        : "memory", "m0", "scc");
}
// Swizzle of K's rows: the 16 rows of one operand read meet different banks.
template <int D>
__device__ __forceinline__ int swizzle_k(int r) {
  return D == 128 ? r & 15 : (r >> 1) & 7;
}

// SLOTS of the ring: 2, or 3 for more than four waves: waves 4 .. are half a tile behind the
// others and keep a third in use.  Two workgroups of four waves fit a CU (hence the bound on
// registers).
template <class T, int D, int SLOTS>
__global__ void __launch_bounds__(SLOTS == 3 ? 64 * kBlockWaves : 256, 2)
    paged_block_kernel(PagedArgs a) {
  constexpr int KS = D / 32, DT = D / 16, NT = kBlockCols / 16;
  constexpr int ROWB = 2 * D;
  constexpr int UNITS = D / 8;
  constexpr int ROWS = 64 / UNITS;         // of one DMA instruction (1 KB)
  constexpr int TILEB = kBlockKeys * ROWB;
  constexpr int V_AT = SLOTS * TILEB;      // K's slots, then V's
  extern __shared__ __align__(256) unsigned char smem[];
  unsigned char* ring = smem;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int waves = __builtin_amdgcn_readfirstlane((int)blockDim.x >> 6);
  int* flag = reinterpret_cast<int*>(ring + 2 * V_AT);  // last tile (+ 1) with a value not finite
  const int col = lane & 15, grp = lane >> 4;
  // XCD-aware order: workgroups go to the XCDs in turn, so XCD x takes a contiguous
  // range, in which the column tiles of one piece of keys meet in its L2.
  uint32_t id;  // (the grid is below 2^31)
  {
    const uint32_t total = gridDim.x, x = blockIdx.x % 8, q8 = total / 8, r8 = total % 8;
    id = x * q8 + min(x, r8) + blockIdx.x / 8;
  }
  const int ct = id % (uint32_t)a.col_tiles;
  id /= (uint32_t)a.col_tiles;
  const int h = id % (uint32_t)a.Hkv;
  id /= (uint32_t)a.Hkv;
  const int part = id % (uint32_t)a.parts;
  const int b = id / (uint32_t)a.parts;
  const int cols = kBlockCols * waves;
  const int n = length_of(a, b), p0 = start_of(a, b, n);
  const Range r = tile_range(a, n, p0, ct * cols, cols);
  const int first = r.start + part * a.part_keys;
  const int last = min(r.end, first + a.part_keys);
  if (part > 0 && first >= r.end) return;
  const int c0 = ct * cols + kBlockCols * wave;   // this wave's columns

  // ---- this lane's columns
  bool padding[NT];
  int lo[NT], hi[NT];
  u32x4_t Q[NT][KS];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int m = c0 + 16 * t + col;
    const bool cok = m < a.M;
    const int pos = p0 + (cok ? m / a.G : 0);
    padding[t] = !cok || pos < 0 || pos >= n;
    lo[t] = hi[t] = 0;
    if (!padding[t]) seen_by(a, n, pos, lo[t], hi[t]);
  }
  f32x4_t O[NT][DT];
  float mx[NT], sum[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    mx[t] = neg_inf();
    sum[t] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) O[t][d] = zero4();
  }
  if (tid == 0) *flag = 0;

  // ---- the stream.  A tile is four pieces of sixteen rows of K and of V, each inside one
  // page.  Waves 0 to 3 bring one each: waves 4 .., which are behind them, have no time to.  A
  // DMA instruction fills ROWS rows (1 KB): lane (row lane / UNITS, unit
  // lane % UNITS) fetches the unit that the swizzle puts there.
  const scalar_ints table = scalars(a.table + b * a.table_stride);
  const int page_mask = (1 << a.page_shift) - 1;
  constexpr int DMAS = 16 / ROWS;
  const int quarter = wave & 3;
  const bool late = SLOTS == 3 && wave >= 4;
  uint32_t k_lane[DMAS], v_lane[DMAS];   // byte offsets (a piece spans < 2^31 bytes)
#pragma unroll
  for (int i = 0; i < DMAS; ++i) {
    const int row = i * ROWS + lane / UNITS;
    k_lane[i] = 2u * (uint32_t)row * (uint32_t)a.k_sr + 16u * ((lane % UNITS) ^ swizzle_k<D>(row));
    v_lane[i] = 2u * (uint32_t)row * (uint32_t)a.v_sr + 16u * ((lane % UNITS) ^ swizzle<D>(row));
  }
  const uint8_t* const k_pool = (const uint8_t*)(a.k + h * a.k_sh);
  const uint8_t* const v_pool = (const uint8_t*)(a.v + h * a.v_sh);
  const int64_t k_page_bytes = 2 * a.k_sp, k_row_bytes = 2 * a.k_sr;
  const int64_t v_page_bytes = 2 * a.v_sp, v_row_bytes = 2 * a.v_sr;
  const uint32_t lds0 = lds_addr(ring);
  const uint32_t k_to = lds0 + quarter * 16 * ROWB, v_to = lds0 + V_AT + quarter * 16 * ROWB;
  auto is_live = [&](int page) { return (uint32_t)page < (uint32_t)a.num_pages; };
  // The wave's rows in the tile at `base`: K's and V's addresses, of page `page`.
  struct Source {
    const uint8_t *k, *v;
  };
  auto source = [&](int base, int page) {
    const uint32_t at = is_live(page) ? page : 0;  // a page that exists; its values are not used
    const uint32_t row = (base + 16 * quarter) & page_mask;
    return Source{k_pool + (at * k_page_bytes + row * k_row_bytes),
                  v_pool + (at * v_page_bytes + row * v_row_bytes)};
  };
  auto bring = [&](const Source& s, uint32_t slot_off) {
    dma_piece(k_to + slot_off, s.k, k_lane);
    dma_piece(v_to + slot_off, s.v, v_lane);
  };
  // The table entry of the wave's rows, read a tile ahead.  (A vector load: a scalar one in
  // flight would turn every wait for LDS into a wait for all of it.)
  const int32_t* const entries = a.table + b * a.table_stride;
  auto entry_for = [&](int base) {
    return entries[max(0, min((base + 16 * quarter) >> a.page_shift, a.table_width - 1))];
  };
  auto page_from = [&](int base, int32_t entry) {
    return (base + 16 * quarter) >> a.page_shift < a.table_width
               ? __builtin_amdgcn_readfirstlane(entry) : -1;
  };

  // Tiles; those from `plain` on up to plain_end are seen whole by every column.  Tile t is
  // in slot (t - plain) mod SLOTS.
  const int tiles = first < last ? (last - first + kBlockKeys - 1) / kBlockKeys : 0;
  const int plain = max(0, r.inner_lo - first + kBlockKeys - 1) / kBlockKeys;
  int plain_end = max(0, min(last, r.inner_hi) - first) / kBlockKeys;
  auto slot_of = [&](int t) {
    return (uint32_t)(t + SLOTS - plain % SLOTS) % (uint32_t)SLOTS * (uint32_t)TILEB;
  };
  int32_t entry = 0;
  if (tiles > 0 && !late) {
    bring(source(first, page_from(first, entry_for(first))), slot_of(0));
    entry = entry_for(first + kBlockKeys);
  }
  // (behind the first tile's DMA: the queries, none for padding, whose values may be anything;
  // and whether an entry of this piece of the table is unmapped, in which case every tile looks)
  bool holes = false;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int m = c0 + 16 * t + col;
    const int qi = m < a.M ? m / a.G : 0, qg = m < a.M ? m - qi * a.G : 0;
    const uint16_t* qp = a.q + b * a.q_sb + qi * a.q_sl + (h * a.G + qg) * a.q_sh + 8 * grp;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Q[t][s] = u32x4_t{0, 0, 0, 0};
      if (!padding[t]) Q[t][s] = *reinterpret_cast<const u32x4_t*>(qp + 32 * s);
    }
  }
  for (int e = (first >> a.page_shift) + lane; e <= (last - 1) >> a.page_shift; e += 64)
    holes |= !is_live(entries[e]);
  holes = __builtin_amdgcn_ballot_w64(holes) != 0;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(Q[t][s]));

  // LDS addresses, slot 0: K's rows of each reduction step, V's of each dim tile (the slot
  // and the row tile are instruction offsets: no vector work between the products)
  uint32_t k_at[KS], v_at[DT];
  {
    const int rt = 4 * grp + (col >> 2);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      k_at[s] = lds0 + ROWB * col + 16u * (uint32_t)((4 * s + grp) ^ swizzle_k<D>(col));
#pragma unroll
    for (int d = 0; d < DT; ++d)
      v_at[d] = lds0 + V_AT + ROWB * rt +
                16u * (uint32_t)((2 * d + ((col >> 1) & 1)) ^ swizzle<D>(rt)) + 8u * (col & 1);
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(k_at[s]));
#pragma unroll
    for (int d = 0; d < DT; ++d) asm volatile("" : "+v"(v_at[d]));
  }
  const float scale = a.scale_log2;
  const bool active = c0 < a.M;            // the wave has columns

  // The pieces of one tile's work; `off`: the slot's offset.
  constexpr int AHEAD = 4;                 // operands in flight
  f32x4_t S[NT][4];
  u32x4_t Pb[NT][2];
  auto scores = [&](uint32_t off) {
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int m = 0; m < 4; ++m) S[c][m] = zero4();
    u32x4_t x[4 * KS];
    auto operand = [&](int o) {  // keys 16 (o & 3) .., dims 32 (o >> 2) ..
      return lds_read16(k_at[o >> 2] + (off + 16 * ROWB * (o & 3)));
    };
#pragma unroll
    for (int o = 0; o < AHEAD; ++o) x[o] = operand(o);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int o = 0; o < 4 * KS; ++o) {
#pragma unroll
      for (int c = 0; c < NT; ++c) S[c][o & 3] = T::mfma(x[o], Q[c][o >> 2], S[c][o & 3]);
      if (o + AHEAD < 4 * KS) x[o + AHEAD] = operand(o + AHEAD);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Weights of column tile c's scores over the maximum `off`, and their sum in this lane.
  auto weigh = [&](int c, float off) {
    float part_sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = exp2_hw(__builtin_fmaf(S[c][2 * k + (i >> 2)][i & 3], scale, -off));
        part_sum[i & 3] += w[i];
      }
      Pb[c][k] = u32x4_t{T::pack(w[0], w[1]), T::pack(w[2], w[3]), T::pack(w[4], w[5]),
                         T::pack(w[6], w[7])};
    }
    return (part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]);
  };
  // The weights are taken over the maximum so far, which need not be the tile's: it moves
  // only when a lane's sixteen weights sum past most_sum, or are not finite (in a
  // part's first tile the maximum is -inf), and then they are taken again.  A maximum per tile
  // would cost a tenth of the vector work.
  constexpr float most_sum = kMostSum * (1 << (int)T::kBlockLift);
  auto softmax = [&] {
    float add[NT];
    bool fits = true;
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      add[c] = weigh(c, mx[c]);
      fits &= add[c] < most_sum;
    }
    if (__builtin_amdgcn_ballot_w64(!fits) != 0) {
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const float to =
            __builtin_fmaxf(mx[c], across4_max(max16_raw(S[c])) * scale - T::kBlockLift);
        const float f = to == neg_inf() ? 1.f : exp2_hw(mx[c] - to);
        mx[c] = to;
        sum[c] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) O[c][d] *= f;
        add[c] = weigh(c, to == neg_inf() ? 0.f : to);
      }
    }
#pragma unroll
    for (int c = 0; c < NT; ++c) sum[c] += add[c];
  };
  auto outputs = [&](uint32_t off) {
    u32x4_t x[2 * DT];
    auto operand = [&](int o) {  // dims 16 (o >> 1) .., keys 32 (o & 1) ..
      const uint32_t ad = v_at[o >> 1] + (off + 32 * ROWB * (o & 1));
      const u32x2_t y0 = read_transposed(ad), y1 = read_transposed(ad + 16u * ROWB);
      return u32x4_t{y0[0], y0[1], y1[0], y1[1]};
    };
#pragma unroll
    for (int o = 0; o < AHEAD; ++o) x[o] = operand(o);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int o = 0; o < 2 * DT; ++o) {
#pragma unroll
      for (int c = 0; c < NT; ++c) O[c][o >> 1] = T::mfma(x[o], Pb[c][o & 1], O[c][o >> 1]);
      if (o + AHEAD < 2 * DT) x[o + AHEAD] = operand(o + AHEAD);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Tile t is there, and its successor, if any, on its way to slot `to`.  (Where that comes from
  // is computed before the barrier, which waves 0 .. mostly wait at.)
  auto arrive = [&](int t, uint32_t to) {
    const int base = first + t * kBlockKeys;
    const bool brings = !late && t + 1 < tiles;
    Source s = {nullptr, nullptr};
    if (brings) s = source(base + kBlockKeys, page_from(base + kBlockKeys, entry));
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (!brings) return;
    bring(s, to);
    entry = entry_for(base + 2 * kBlockKeys);
  };

  // Any tile: masks, rows nobody sees, unmapped pages, the last.
  auto live_at = [&](int base, int i) {
    return !holes || is_live(page_at(a, table, base + 16 * i));
  };
  auto edge_tile = [&](int t) {
    const uint32_t off = slot_of(t);
    const int base = first + t * kBlockKeys;
    arrive(t, slot_of(t + 1));
    // V rows that no column sees become zeros; values that are not finite
    // are taken out where some columns see them and others do not (which must not get
    // 0 x inf) and added one by one below.
    const bool uneven = is_uneven(r, base, kBlockKeys);
    bool odd = false;
    for (int x = tid; x < kBlockKeys * UNITS; x += 64 * waves) {
      const int key = base + x / UNITS;
      u32x4_t* at = reinterpret_cast<u32x4_t*>(ring + V_AT + off + 16 * x);
      bool lv = true;
      if (holes) {
        const int e = key >> a.page_shift;  // (a vector load: rows differ between lanes)
        lv = e < a.table_width && is_live(entries[e]);
      }
      if (!lv || key < r.lo || key >= r.end) {
        *at = u32x4_t{0, 0, 0, 0};
        continue;
      }
      if (!uneven) continue;
      u32x4_t v = *at;
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool b0 = (v[e] & T::kExp) == T::kExp, b1 = ((v[e] >> 16) & T::kExp) == T::kExp;
        bad |= b0 || b1;
        if (b0) v[e] &= 0xffff0000u;
        if (b1) v[e] &= 0x0000ffffu;
      }
      if (bad) *at = v;
      odd |= bad;
    }
    if (odd) *flag = t + 1;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const bool dirty = *(const volatile __attribute__((address_space(3))) int*)flag == t + 1;
    if (!active) return;
    scores(off);
    const bool live[4] = {live_at(base, 0), live_at(base, 1), live_at(base, 2), live_at(base, 3)};
    uint32_t seen[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      seen[c] = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = base + 16 * (i >> 2) + 4 * grp + (i & 3);
        const bool ok = live[i >> 2] && key >= lo[c] && key < hi[c];
        if (ok) seen[c] |= 1u << i;
        S[c][i >> 2][i & 3] = ok ? S[c][i >> 2][i & 3] : neg_inf();
      }
    }
    softmax();
    outputs(off);
    if (!dirty) return;
    const args_again_t z = args_again();
    for (int kk = 0; kk < kBlockKeys; ++kk) {
      const int key = base + kk;
      if (!live_at(base, kk >> 4) || key < r.lo || key >= r.end) continue;
      const int from = 16 * ((kk & 15) >> 2) + col, slot_i = 4 * (kk >> 4) + (kk & 3);
      const uint16_t* vp = z->v + h * z->v_sh + page_at(a, table, key) * z->v_sp +
                           (int64_t)(key & page_mask) * z->v_sr;
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const bool ok = (__shfl(seen[c], from, 64) >> slot_i) & 1;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = vp[16 * d + 4 * grp + e];
            if (ok && (x & T::kExp) == T::kExp) O[c][d][e] += T::value(x);
          }
      }
    }
  };
  // Edge tiles, then the plain ones (every column sees all of the tile), then edge
  // tiles: two passes of a loop, so that the edge code is there once.
  // Waves 4 .. share their SIMDs with waves 0 .. and go half a tile behind them: their
  // softmax runs while the others' products do.
  if (holes) plain_end = 0;
  int t = 0;
  // A plain tile in slot SLOT (constants, so that no address is computed); false: the last.
  auto plain_tile = [&](auto slot) {
    constexpr uint32_t off = decltype(slot)::value * TILEB;
    constexpr uint32_t after = (decltype(slot)::value + 2) % SLOTS * TILEB;
    const bool more = t + 1 < plain_end;
    if (active) scores(off);
    if (late && more) arrive(t + 1, after);
    __builtin_amdgcn_sched_barrier(0);
    if (active) {
      softmax();
      __builtin_amdgcn_sched_barrier(0);
      outputs(off);
    }
    ++t;
    if (!late && more) arrive(t, after);
    return more;
  };
  for (int pass = 0; pass < 2; ++pass) {
    for (const int to = pass == 0 && plain < plain_end ? plain : tiles; t < to; ++t) edge_tile(t);
    if (t >= plain_end) continue;
    arrive(t, TILEB);
    for (;;) {
      if (!plain_tile(std::integral_constant<int, 0>{})) break;
      if (!plain_tile(std::integral_constant<int, 1>{})) break;
      if constexpr (SLOTS == 3)
        if (!plain_tile(std::integral_constant<int, 2>{})) break;
    }
  }

  // ---- out: lane (col, grp) holds dims 16 d + 4 grp .. of its columns
  const args_again_t z = args_again();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int m = c0 + 16 * t + col;
    float total = across4_sum(sum[t]);
    if (padding[t]) {  // (its scores were not masked in tiles that every row sees)
      mx[t] = neg_inf();
      total = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) O[t][d] = zero4();
    }
    if (m >= z->M) continue;
    if (z->parts > 1) {
      const int64_t at = (((int64_t)b * z->Hkv + h) * z->M + m) * z->parts + part;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        *reinterpret_cast<f32x4_t*>(z->part_out + at * D + 16 * d + 4 * grp) = O[t][d];
      if (grp == 0) {
        z->part_ml[2 * at] = mx[t];
        z->part_ml[2 * at + 1] = total;
      }
      continue;
    }
    const int qi = m / z->G;
    const int64_t row = ((int64_t)b * z->Lq + qi) * z->Hq + h * z->G + (m - qi * z->G);
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      u32x2_t o = {0u, 0u};
      if (total != 0.f)
        o = u32x2_t{T::pack(O[t][d][0] * inv, O[t][d][1] * inv),
                    T::pack(O[t][d][2] * inv, O[t][d][3] * inv)};
      *reinterpret_cast<u32x2_t*>(z->out + row * D + 16 * d + 4 * grp) = o;
    }
    if (grp == 0) z->lse[row] = total == 0.f ? neg_inf() : kLn2 * (mx[t] + log2_hw(total));
  }
}

// Joining: WAVES waves per column; each reads all of the column's maxima and sums,
// and the outputs of every WAVES-th part, eight rows in flight.
template <class T, int D, int WAVES>
__global__ void __launch_bounds__(256) paged_join_kernel(PagedArgs a) {
  constexpr int COLS = 4 / WAVES;               // columns of a workgroup
  constexpr int VALUES = D / 64;                // dims of a lane
  typedef float vec_t __attribute__((ext_vector_type(VALUES)));
  __shared__ vec_t acc_l[256];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t columns = (uint32_t)a.B * a.Hkv * a.M;       // (at most 2^31 - 1)
  const uint32_t c_raw = blockIdx.x * COLS + wave / WAVES;    // (b Hkv + h) M + m
  const bool there = c_raw < columns;
  const int64_t c = there ? c_raw : columns - 1;
  const uint32_t bh = (uint32_t)c / (uint32_t)a.M;
  const int m = (uint32_t)c - bh * a.M;
  const int b = bh / (uint32_t)a.Hkv, h = bh % (uint32_t)a.Hkv;
  const int n = length_of(a, b);
  const Range r = tile_range(a, n, start_of(a, b, n), m / a.tile_cols * a.tile_cols, a.tile_cols);
  const int np = max(1, (r.end - r.start + a.part_keys - 1) / a.part_keys);
  const float* ml = a.part_ml + 2 * c * a.parts;
  const vec_t* po = reinterpret_cast<const vec_t*>(a.part_out + c * a.parts * D) + lane;
  vec_t v[8];
  float w[8];
  auto fetch = [&](int p0) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {  // (a part past the last is the last one, and not added)
      const int p = min(p0 + u * WAVES, np - 1);
      v[u] = po[(int64_t)p * 64];
      w[u] = ml[2 * p];
    }
  };
  fetch(wave % WAVES);
  float M = neg_inf();
  for (int p = lane; p < np; p += 64) M = __builtin_fmaxf(M, ml[2 * p]);
  M = wave_max(M);
  float total = 0.f;
  for (int p = lane; p < np; p += 64)
    total += (M == neg_inf() ? 1.f : exp2_hw(ml[2 * p] - M)) * ml[2 * p + 1];
  total = wave_sum(total);
  vec_t acc = {};
  for (int p0 = wave % WAVES;;) {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (p0 + u * WAVES < np) acc += (M == neg_inf() ? 1.f : exp2_hw(w[u] - M)) * v[u];
    p0 += 8 * WAVES;
    if (p0 >= np) break;
    fetch(p0);
  }
  if constexpr (WAVES > 1) {
    acc_l[threadIdx.x] = acc;
    __syncthreads();
    if (wave % WAVES != 0) return;
#pragma unroll
    for (int x = 1; x < WAVES; ++x) acc += acc_l[threadIdx.x + 64 * x];
  }
  if (!there) return;
  const int i = m / a.G;
  const int64_t row = ((int64_t)b * a.Lq + i) * a.Hq + h * a.G + (m - i * a.G);
  const float inv = total == 0.f ? 0.f : 1.f / total;
  uint16_t* out = a.out + row * D + VALUES * lane;
  if constexpr (VALUES == 2)
    *reinterpret_cast<uint32_t*>(out) = total == 0.f ? 0u : T::pack(acc[0] * inv, acc[1] * inv);
  else
    *out = total == 0.f ? 0 : (uint16_t)T::pack(acc[0] * inv, 0.f);
  if (lane == 0) a.lse[row] = total == 0.f ? neg_inf() : kLn2 * (M + log2_hw(total));
}

// Columns of a workgroup: up to 16 the streaming kernel; more, whole waves of the
// block kernel, four at least (each brings its share of the rows), as even as they come.
int columns_of(int64_t M) {
  if (M <= 16) return 16;
  const int64_t groups = (M + kBlockCols - 1) / kBlockCols;
  const int64_t tiles = (groups + kBlockWaves - 1) / kBlockWaves;
  return (int)std::max<int64_t>(4, (groups + tiles - 1) / tiles) * kBlockCols;
}

// Most keys that the columns of one workgroup can see.  (Rows at the end of their
// sequence have at most the other rows behind them.)
int64_t span_bound(int64_t max_len, int64_t q_len, int64_t group, int64_t cols, int64_t window,
                   int causal, bool at_end) {
  if (window < 0) return max_len;
  const int64_t rows = std::min<int64_t>(q_len, cols / group + 2);
  const int64_t right = causal ? 0 : at_end ? std::min(window, q_len) : window;
  return std::min(max_len, rows + window + right + 1);
}

template <class T, int D>
int launch(const PagedArgs& a, hipStream_t stream) {
  const int64_t grid = (int64_t)a.B * a.Hkv * a.col_tiles * a.parts;
  const int64_t cols = (int64_t)a.B * a.Hkv * a.M;
  const int64_t threads = a.tile_cols == 16 ? 64 * kWaves : 64 * a.tile_cols / kBlockCols;
  // (a launch holds fewer than 2^32 threads; the join has 64 a column, or 256 of at most 1024)
  if (grid > 0xffffffffll / threads || (a.parts > 1 && cols > (1 << 26) - 4) || cols > 0x7fffffff)
    return MRSA_ERR_UNSUPPORTED;
  if (a.tile_cols == 16) {
    static_assert(kStreamLds >= kWaves * std::max(kTile * 2 * D, 16 * (D + 4) * 4));
    hipLaunchKernelGGL((paged_attn_kernel<T, D>), dim3((unsigned)grid), dim3(64 * kWaves),
                       kStreamLds, stream, a);
  } else {
    const int waves = a.tile_cols / kBlockCols;
    auto kern = waves > 4 ? paged_block_kernel<T, D, 3> : paged_block_kernel<T, D, 2>;
    const size_t lds = (waves > 4 ? 3 : 2) * 2 * kBlockKeys * 2 * D + 16;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                            hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
      return MRSA_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * waves), lds, stream, a);
  }
  int st = mrsa_launch_status();
  if (st != MRSA_OK || a.parts == 1) return st;
  // Four waves per column where there are many parts and few columns, otherwise one. Both
  // kernels' time by four and by one: 28 columns of 64 parts 11.0 and 12.7 us, 448 of 64 20.3 and
  // 22.4, 896 of 32 23.2 and 24.2, of 12 20.6 and 19.3, 2688 of 12 27.4 and 23.7.
  if (a.parts > 16 && cols <= 1024)
    hipLaunchKernelGGL((paged_join_kernel<T, D, 4>), dim3((unsigned)cols), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_join_kernel<T, D, 1>), dim3((unsigned)((cols + 3) / 4)), dim3(256), 0,
                       stream, a);
  return mrsa_launch_status();
}

}  // namespace

extern "C" int64_t mrsa_paged_attention_workspace_bytes(int64_t batch, int64_t q_len,
                                                        int64_t q_heads, int64_t head_dim,
                                                        int64_t parts) {
  const int64_t most = 1ll << 31;
  if (batch < 0 || q_len < 0 || q_heads <= 0 || head_dim <= 0 || parts < 1 || batch > most ||
      q_len > most || q_heads > 65536 || head_dim > 4096 || parts > kMaxParts)
    return -1;
  if (parts == 1 || batch == 0 || q_len == 0) return 0;
  if (q_len > (1ll << 38) / batch / q_heads) return -1;   // (so that the product fits 63 bits)
  return batch * q_len * q_heads * parts * (head_dim + 2) * (int64_t)sizeof(float);
}

extern "C" int mrsa_paged_attention_fwd(
    const void* q, int64_t q_batch_stride, int64_t q_row_stride, int64_t q_head_stride,
    const void* k_pages, int64_t k_page_stride, int64_t k_slot_stride, int64_t k_head_stride,
    const void* v_pages, int64_t v_page_stride, int64_t v_slot_stride, int64_t v_head_stride,
    const int32_t* page_table, int64_t page_table_stride, int64_t table_pages, int64_t num_pages,
    int64_t page_size, const int32_t* cache_lens, const int32_t* query_starts, int64_t max_len,
    int64_t batch, int64_t q_len, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
    int32_t dtype, int32_t causal,
    int64_t window, float sm_scale, int64_t parts, void* workspace, int64_t workspace_bytes,
    void* out, float* lse, void* stream) {
  if (batch < 0 || q_len < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 ||
      max_len < 0 || table_pages < 0 || num_pages < 0 || page_size <= 0 || parts < 1 ||
      parts > kMaxParts)
    return MRSA_ERR_INVALID_ARGUMENT;
  if (!(sm_scale > 0.f) || !(sm_scale * kLog2e < __builtin_inff()))
    return MRSA_ERR_INVALID_ARGUMENT;
  if (dtype != MRSA_DTYPE_BF16 && dtype != MRSA_DTYPE_FP16) return MRSA_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return MRSA_ERR_UNSUPPORTED;
  if ((page_size & (page_size - 1)) != 0 || page_size < 16 || page_size > (1 << 20))
    return MRSA_ERR_UNSUPPORTED;
  const int64_t most = kFar;
  if (max_len >= most || q_len >= most || table_pages >= most || num_pages > 0x7fffffff ||
      batch > most || q_heads > 65536 || (q_len > 0 && q_heads / kv_heads > most / q_len))
    return MRSA_ERR_UNSUPPORTED;
  if (batch == 0 || q_len == 0) return MRSA_OK;
  if (!q || !cache_lens || !out || !lse) return MRSA_ERR_INVALID_ARGUMENT;
  if (table_pages == 0 || num_pages == 0) max_len = 0;   // no keys anywhere
  else if (!page_table || !k_pages || !v_pages) return MRSA_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out) % 16 != 0 ||
      (q_batch_stride | q_row_stride | q_head_stride | k_page_stride | k_slot_stride |
       k_head_stride | v_page_stride | v_slot_stride | v_head_stride) % 8 != 0)
    return MRSA_ERR_UNSUPPORTED;
  if (k_slot_stride < 0 || k_slot_stride >= (1 << 26) || v_slot_stride < 0 ||
      v_slot_stride >= (1 << 26))
    return MRSA_ERR_UNSUPPORTED;
  const int64_t need = mrsa_paged_attention_workspace_bytes(batch, q_len, q_heads, head_dim, parts);
  if (need < 0) return MRSA_ERR_UNSUPPORTED;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16 != 0))
    return MRSA_ERR_INVALID_ARGUMENT;
  PagedArgs a = {};
  a.q = (const uint16_t*)q;
  a.q_sb = q_batch_stride, a.q_sl = q_row_stride, a.q_sh = q_head_stride;
  a.k = (const uint16_t*)k_pages;
  a.k_sp = k_page_stride, a.k_sr = k_slot_stride, a.k_sh = k_head_stride;
  a.v = (const uint16_t*)v_pages;
  a.v_sp = v_page_stride, a.v_sr = v_slot_stride, a.v_sh = v_head_stride;
  a.table = page_table;
  a.table_stride = page_table_stride;
  a.table_width = (int)table_pages;
  a.page_shift = __builtin_ctzll((uint64_t)page_size);
  a.num_pages = (int)num_pages;
  a.lens = cache_lens;
  a.starts = query_starts;
  a.max_len = (int)max_len;
  a.B = (int)batch, a.Lq = (int)q_len, a.Hq = (int)q_heads, a.Hkv = (int)kv_heads;
  a.G = (int)(q_heads / kv_heads);
  a.M = a.Lq * a.G;
  a.causal = causal != 0;
  a.window = window < 0 ? -1 : (int)std::min<int64_t>(window, most);
  a.scale_log2 = sm_scale * kLog2e;
  a.parts = (int)parts;
  a.tile_cols = columns_of(a.M);
  a.col_tiles = (a.M + a.tile_cols - 1) / a.tile_cols;
  const int64_t span =
      span_bound(max_len, q_len, a.G, a.tile_cols, a.window, a.causal, !query_starts) +
      (a.window >= 0 ? kTile - 1 : 0);  // (a window's first tile may start before it)
  const int64_t step = a.tile_cols == 16 ? kStep : kBlockKeys;
  // (at least one step: without keys, max_len 0, the join still divides by it)
  a.part_keys = (int)((std::max<int64_t>(1, (span + parts - 1) / parts) + step - 1) / step * step);
  a.out = (uint16_t*)out;
  a.lse = lse;
  a.part_out = (float*)workspace;
  if (parts > 1) a.part_ml = a.part_out + batch * q_len * q_heads * parts * head_dim;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MRSA_DTYPE_BF16)
    return head_dim == 128 ? launch<Bf16, 128>(a, s) : launch<Bf16, 64>(a, s);
  return head_dim == 128 ? launch<Fp16, 128>(a, s) : launch<Fp16, 64>(a, s);
}
