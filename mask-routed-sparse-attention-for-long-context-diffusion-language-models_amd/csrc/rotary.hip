// Rotary positions of query and key heads, and the same rotation fused with
// the write of new rows into the pages of a K/V cache.
//
// A head's first 2 `half` dims hold pairs (x1, x2): dims i and i + half (half
// layout) or 2 i and 2 i + 1 (interleaved).  With c, s = cos, sin of row
// `position` of the tables:
//     y1 = x1 c - x2 s,   y2 = x2 c + x1 s          (inverse: s -> -s,
// the transpose, which is the gradient).  Dims past 2 half are copied.
// Products and sums are fp32 with fp32 tables, rounded once to the tensors'
// type.  A position outside the tables gives NaN rows: nothing is read there.
//
// Pure streams: every element is read once and written once, so the kernels
// are bound by HBM for long inputs and by the launch for short ones.  A thread
// takes one 16-byte unit (or the two units of a half-layout pair) of up to
// kHeadsPerThread heads of one token, so that a token's table row is read once
// per thread and not once per head, and all its loads are in flight together.
// 28 + 4 heads of 128 dims, bf16: 16384 rows (273 MB) 47-54 us, 5.0-5.8 TB/s (a large
// copy, whose results do not fit the caches: 5.3); 32 rows 3.5 us, a launch.  Append of 16002
// rows of 28 + 4 + 4 heads (292 MB) 53 us; of 16 rows 4.2 us.
#include "mrsa_device.h"

using namespace mrsa;

namespace {

constexpr int kThreads = 256;
constexpr int kMostThreads = 512;
constexpr int kHeadsPerThread = 4;
constexpr int kScalarHeads = 8;
// Head units from which a thread takes that many.  Half as many units (512 rows of 32 heads):
// 4.35 us, 3.86 by a head each; as many: 4.99 and 5.17; twice: 7.03 and 7.81.
constexpr int64_t kManyUnits = 256 * 1024;

// One stream of heads: [batch, row, head] strides in elements, last dim dense.
struct Heads {
  const void* src;
  int64_t sb, sl, sh;
  void* dst;          // paged: the page pool
  int64_t db, dl, dh; // paged: page, row, head strides
  int heads;
};

struct RotaryArgs {
  Heads q, k, v;
  const float* cos_t;
  const float* sin_t;
  int64_t table_rows;
  const int64_t* positions;  // optional
  int64_t ps_b, ps_l;
  int tokens, L;             // tokens = batch * L
  int D, half;
  float sign;                // -1: inverse
  // paged writes of k and v
  const int64_t* slots;
  int64_t sl_b, sl_l;
  const int32_t* table;
  int64_t table_stride;
  int table_width, page_shift;
  int64_t num_pages;
  int units, head_slots, tokens_per_block;
};

template <class T>
struct Traits;
template <>
struct Traits<__bf16> {
  static constexpr int kPer16 = 8;
};
template <>
struct Traits<_Float16> {
  static constexpr int kPer16 = 8;
};
template <>
struct Traits<float> {
  static constexpr int kPer16 = 4;
};

template <class T>
struct alignas(16) Vec {
  T e[Traits<T>::kPer16];
};

// Page and row of token (b, l); false if the token has no place.
template <class T, bool PAGED>
__device__ __forceinline__ bool cache_row(const RotaryArgs& a, int b, int l, int64_t& page,
                                          int64_t& row) {
  const int64_t slot = a.slots[b * a.sl_b + l * a.sl_l];
  if (slot < 0 || (slot >> a.page_shift) >= a.table_width) return false;
  const int32_t p = a.table[b * a.table_stride + (slot >> a.page_shift)];
  if (p < 0 || p >= a.num_pages) return false;
  page = p;
  row = slot & ((1ll << a.page_shift) - 1);
  return true;
}

// One pair; the order of the roundings is fixed, so that every kernel here gives
// the same bits.
__device__ __forceinline__ void turn_pair(float& x1, float& x2, float c, float s) {
  const float y1 = __builtin_fmaf(x1, c, -__fmul_rn(x2, s));
  x2 = __builtin_fmaf(x2, c, __fmul_rn(x1, s));
  x1 = y1;
}

template <class T, bool INTERLEAVED>
__device__ __forceinline__ void turn(Vec<T>& x, Vec<T>& y, const float* c, const float* s) {
  constexpr int E = Traits<T>::kPer16;
  if constexpr (INTERLEAVED) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      float x1 = (float)x.e[2 * i], x2 = (float)x.e[2 * i + 1];
      turn_pair(x1, x2, c[i], s[i]);
      x.e[2 * i] = (T)x1;
      x.e[2 * i + 1] = (T)x2;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float x1 = (float)x.e[i], x2 = (float)y.e[i];
      turn_pair(x1, x2, c[i], s[i]);
      x.e[i] = (T)x1;
      y.e[i] = (T)x2;
    }
  }
}

// The stream, place and rows of one head out of q, k and (paged) v.  Fields are
// selected value by value: a pointer into the arguments would put them in
// scratch memory.
template <class T, bool PAGED>
struct Rows {
  const T *q_in, *k_in, *v_in;
  T *q_out, *k_out, *v_out;
  bool placed;

  __device__ __forceinline__ Rows(const RotaryArgs& a, int b, int l) {
    q_in = (const T*)a.q.src + b * a.q.sb + l * a.q.sl;
    k_in = (const T*)a.k.src + b * a.k.sb + l * a.k.sl;
    q_out = (T*)a.q.dst + b * a.q.db + l * a.q.dl;
    placed = true;
    if constexpr (PAGED) {
      int64_t page = 0, row = 0;
      placed = cache_row<T, PAGED>(a, b, l, page, row);
      v_in = (const T*)a.v.src + b * a.v.sb + l * a.v.sl;
      k_out = (T*)a.k.dst + page * a.k.db + row * a.k.dl;
      v_out = (T*)a.v.dst + page * a.v.db + row * a.v.dl;
    } else {
      k_out = (T*)a.k.dst + b * a.k.db + l * a.k.dl;
    }
  }
  // Head h of all; `turns`: q and k heads, `there`: it has a place to go.
  __device__ __forceinline__ void head(const RotaryArgs& a, int h, const T*& in, T*& out,
                                       bool& turns, bool& there) const {
    const bool is_q = h < a.q.heads;
    const bool is_v = PAGED && h >= a.q.heads + a.k.heads;
    int hh = is_q ? h : h - a.q.heads;
    in = is_q ? q_in : k_in;
    out = is_q ? q_out : k_out;
    int64_t sh = is_q ? a.q.sh : a.k.sh, dh = is_q ? a.q.dh : a.k.dh;
    if constexpr (PAGED) {
      hh = is_v ? hh - a.k.heads : hh;
      in = is_v ? v_in : in;
      out = is_v ? v_out : out;
      sh = is_v ? a.v.sh : sh;
      dh = is_v ? a.v.dh : dh;
    }
    in += hh * sh;
    out += hh * dh;
    turns = !is_v;
    there = is_q || placed;
  }
};

// Appended rows are stored past the caches (evicted first): 16002 rows of 28 + 4 + 4
// heads take 53 us so and 58 without.  The dense rotation, whose result the next kernel reads,
// leaves it there: 16384 rows 54 us, 51 past the caches; short ones alike.
template <bool PAST, class T>
__device__ __forceinline__ void store(T* to, const Vec<T>& v) {
  u32x4_t* at = reinterpret_cast<u32x4_t*>(to);
  if constexpr (PAST)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, v), at);
  else
    *at = __builtin_bit_cast(u32x4_t, v);
}

// 16-byte units; PAGED: k and v go to pages (v is copied), else only q and k.
// HEADS: heads of a thread.
template <class T, bool INTERLEAVED, bool PAGED, int HEADS>
__global__ void __launch_bounds__(kMostThreads) rotary_kernel(RotaryArgs a) {
  constexpr int E = Traits<T>::kPer16;
  constexpr int TN = INTERLEAVED ? E / 2 : E;  // table values of a unit
  const int per_token = a.units * a.head_slots;
  const int total_heads = a.q.heads + a.k.heads + (PAGED ? a.v.heads : 0);
  const int rot_units = a.half / TN;
  const int tail_at = 2 * a.half;
  for (int lid = threadIdx.x; lid < a.tokens_per_block * per_token; lid += blockDim.x) {
    const int ti = lid / per_token;
    const int64_t tok = (int64_t)blockIdx.x * a.tokens_per_block + ti;
    if (tok >= a.tokens) return;
    const int rem = lid - ti * per_token;
    const int hs = rem / a.units;
    const int u = rem - hs * a.units;
    const int b = (int)tok / a.L, l = (int)tok - b * a.L;
    const Rows<T, PAGED> rows(a, b, l);
    const bool rotate = u < rot_units;
    // dims of this unit: [at, at + E) and, half layout, [at2, at2 + E)
    const int at = rotate ? u * E : tail_at + (u - rot_units) * E;
    const int at2 = at + a.half;
    const bool two = !INTERLEAVED && rotate;
    Vec<T> x[HEADS], y[HEADS];
    T* out[HEADS];
    bool turns[HEADS], there[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int h = hs + i * a.head_slots;
      const T* in;
      rows.head(a, min(h, total_heads - 1), in, out[i], turns[i], there[i]);
      there[i] &= h < total_heads;
      x[i] = *reinterpret_cast<const Vec<T>*>(in + at);
      if (two) y[i] = *reinterpret_cast<const Vec<T>*>(in + at2);
    }
    float c[TN], s[TN];
    if (rotate) {
      const int64_t pos = a.positions ? a.positions[b * a.ps_b + l * a.ps_l] : l;
      if (pos >= 0 && pos < a.table_rows) {
        const float* cp = a.cos_t + pos * a.half + u * TN;
        const float* sp = a.sin_t + pos * a.half + u * TN;
        if constexpr (TN >= 4) {
#pragma unroll
          for (int i = 0; i < TN / 4; ++i) {
            const f32x4_t cv = reinterpret_cast<const f32x4_t*>(cp)[i];
            const f32x4_t sv = reinterpret_cast<const f32x4_t*>(sp)[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) c[4 * i + j] = cv[j], s[4 * i + j] = a.sign * sv[j];
          }
        } else {
          const f32x2_t cv = *reinterpret_cast<const f32x2_t*>(cp);
          const f32x2_t sv = *reinterpret_cast<const f32x2_t*>(sp);
#pragma unroll
          for (int j = 0; j < 2; ++j) c[j] = cv[j], s[j] = a.sign * sv[j];
        }
      } else {
#pragma unroll
        for (int i = 0; i < TN; ++i) c[i] = s[i] = __builtin_nanf("");
      }
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      if (!there[i]) continue;
      if (rotate && turns[i]) turn<T, INTERLEAVED>(x[i], y[i], c, s);
      store<PAGED>(out[i] + at, x[i]);
      if (two) store<PAGED>(out[i] + at2, y[i]);
    }
  }
}

// The same one value (a tail dim) or pair at a time, for head parts that 16-byte
// units do not divide and for unaligned tensors: units = half pairs and D - 2 half
// tail dims, of kScalarHeads heads a thread.  Bound by the number of its loads and stores:
// 16384 rows of 28 + 4 heads 63 us, 49 by 16-byte units (161 with a head a thread); 32 rows 4.7
// and 4.1.
template <class T, bool INTERLEAVED, bool PAGED>
__global__ void __launch_bounds__(kThreads) rotary_scalar_kernel(RotaryArgs a) {
  const int per_token = a.units * a.head_slots;
  const int total_heads = a.q.heads + a.k.heads + (PAGED ? a.v.heads : 0);
  for (int lid = threadIdx.x; lid < a.tokens_per_block * per_token; lid += kThreads) {
    const int ti = lid / per_token;
    const int64_t tok = (int64_t)blockIdx.x * a.tokens_per_block + ti;
    if (tok >= a.tokens) return;
    const int rem = lid - ti * per_token;
    const int hs = rem / a.units;
    const int u = rem - hs * a.units;
    const int b = (int)tok / a.L, l = (int)tok - b * a.L;
    const Rows<T, PAGED> rows(a, b, l);
    const bool pair = u < a.half;
    const int i1 = !pair ? u + a.half : INTERLEAVED ? 2 * u : u;
    const int i2 = !pair ? i1 : INTERLEAVED ? 2 * u + 1 : u + a.half;
    T x1[kScalarHeads], x2[kScalarHeads];
    T* out[kScalarHeads];
    bool turned[kScalarHeads], there[kScalarHeads];
#pragma unroll
    for (int i = 0; i < kScalarHeads; ++i) {
      const int h = hs + i * a.head_slots;
      const T* in;
      rows.head(a, min(h, total_heads - 1), in, out[i], turned[i], there[i]);
      there[i] &= h < total_heads;
      x1[i] = in[i1];
      x2[i] = in[i2];
    }
    float c = __builtin_nanf(""), s = c;
    if (pair) {
      const int64_t pos = a.positions ? a.positions[b * a.ps_b + l * a.ps_l] : l;
      if (pos >= 0 && pos < a.table_rows) {
        c = a.cos_t[pos * a.half + u];
        s = a.sign * a.sin_t[pos * a.half + u];
      }
    }
#pragma unroll
    for (int i = 0; i < kScalarHeads; ++i) {
      if (!there[i]) continue;
      if (pair && turned[i]) {
        float f1 = (float)x1[i], f2 = (float)x2[i];
        turn_pair(f1, f2, c, s);
        x1[i] = (T)f1;
        x2[i] = (T)f2;
      }
      out[i][i1] = x1[i];
      if (pair) out[i][i2] = x2[i];
    }
  }
}

template <class T, bool PAGED>
int launch(RotaryArgs a, bool interleaved, hipStream_t stream) {
  constexpr int E = Traits<T>::kPer16;
  const int heads = a.q.heads + a.k.heads + (PAGED ? a.v.heads : 0);
  // 16-byte units need whole units of pairs and of tail dims, and every row aligned.
  bool vec = a.D % E == 0 && (interleaved ? 2 * a.half : a.half) % E == 0 &&
             ((uintptr_t)a.cos_t | (uintptr_t)a.sin_t) % 16 == 0;
  const Heads* segs[3] = {&a.q, &a.k, &a.v};
  for (const Heads* s : segs) {
    if (s->heads == 0) continue;
    vec = vec && ((uintptr_t)s->src | (uintptr_t)s->dst) % 16 == 0 &&
          (s->sb | s->sl | s->sh | s->db | s->dl | s->dh) % E == 0;
  }
  int heads_each = 1;
  if (vec) {
    const int rot = a.half / (interleaved ? E / 2 : E);
    a.units = rot + (a.D - 2 * a.half) / E;
    // Few tokens: a head per thread, so that as many threads as there are work; many: the
    // table row of a thread serves kHeadsPerThread heads.
    const int64_t one = (int64_t)a.tokens * heads * a.units;
    if (one >= kManyUnits) heads_each = kHeadsPerThread;
    a.head_slots = (heads + heads_each - 1) / heads_each;
  } else {
    a.units = a.D - a.half;
    a.head_slots = (heads + kScalarHeads - 1) / kScalarHeads;
  }
  const int per_token = a.units * a.head_slots;
  a.tokens_per_block = std::max(1, kThreads / per_token);
  // The block size that whole tokens fill best: 36 heads of 128 dims make 72 threads a
  // token, seven tokens 504 of 512 threads (three 216 of 256: 6% slower).
  int threads = kThreads;
  if (vec) {
    int waste = 64;  // of each 64 threads
    for (int t = a.tokens_per_block; t * per_token <= kMostThreads; ++t) {
      const int whole = (t * per_token + 63) / 64 * 64;
      const int idle = 64 * (whole - t * per_token) / whole;
      if (whole >= kThreads && idle < waste) waste = idle, a.tokens_per_block = t, threads = whole;
    }
    if (per_token > kMostThreads) {  // a token takes several even rounds
      const int rounds = (per_token + kMostThreads - 1) / kMostThreads;
      threads = ((per_token + rounds - 1) / rounds + 63) / 64 * 64;
    }
  }
  const int64_t blocks = ((int64_t)a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  if (blocks > 0xffffffffll / threads) return MRSA_ERR_UNSUPPORTED;  // (threads of a launch)
  void (*kern)(RotaryArgs);
  if (!vec)
    kern = interleaved ? rotary_scalar_kernel<T, true, PAGED>
                       : rotary_scalar_kernel<T, false, PAGED>;
  else if (heads_each == 1)
    kern = interleaved ? rotary_kernel<T, true, PAGED, 1> : rotary_kernel<T, false, PAGED, 1>;
  else
    kern = interleaved ? rotary_kernel<T, true, PAGED, kHeadsPerThread>
                       : rotary_kernel<T, false, PAGED, kHeadsPerThread>;
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(threads), 0, stream, a);
  return mrsa_launch_status();
}

template <bool PAGED>
int dispatch(const RotaryArgs& a, int dtype, int interleaved, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case MRSA_DTYPE_BF16: return launch<__bf16, PAGED>(a, interleaved != 0, s);
    case MRSA_DTYPE_FP16: return launch<_Float16, PAGED>(a, interleaved != 0, s);
    case MRSA_DTYPE_FP32: return launch<float, PAGED>(a, interleaved != 0, s);
    default: return MRSA_ERR_INVALID_ARGUMENT;
  }
}

// What both entry points check of the sizes; 0 tokens or heads pass.
bool sizes_ok(int64_t batch, int64_t seq_len, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
              int64_t rotary_dim, int64_t table_rows) {
  return batch >= 0 && seq_len >= 0 && q_heads >= 0 && kv_heads >= 0 && head_dim > 0 &&
         rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim && table_rows >= 0;
}
bool sizes_fit(int64_t batch, int64_t seq_len, int64_t q_heads, int64_t kv_heads,
               int64_t head_dim) {
  const int64_t most = 0x7fffffff;
  if (batch > most || seq_len > most || q_heads > 65536 || kv_heads > 65536 || head_dim > 4096)
    return false;
  return batch == 0 || seq_len <= most / batch;
}

}  // namespace

extern "C" int mrsa_rotary_fwd(const void* q, int64_t q_batch_stride, int64_t q_row_stride,
                               int64_t q_head_stride, const void* k, int64_t k_batch_stride,
                               int64_t k_row_stride, int64_t k_head_stride,
                               const float* cos_table, const float* sin_table, int64_t table_rows,
                               const int64_t* positions, int64_t positions_batch_stride,
                               int64_t positions_row_stride, int64_t batch, int64_t seq_len,
                               int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                               int64_t rotary_dim, int32_t dtype, int32_t interleaved,
                               int32_t inverse, void* q_out, void* k_out, void* stream) {
  if (!sizes_ok(batch, seq_len, q_heads, kv_heads, head_dim, rotary_dim, table_rows))
    return MRSA_ERR_INVALID_ARGUMENT;
  if (dtype < MRSA_DTYPE_BF16 || dtype > MRSA_DTYPE_FP32) return MRSA_ERR_INVALID_ARGUMENT;
  if (!sizes_fit(batch, seq_len, q_heads, kv_heads, head_dim)) return MRSA_ERR_UNSUPPORTED;
  if (batch * seq_len == 0 || q_heads + kv_heads == 0) return MRSA_OK;
  if ((q_heads && (!q || !q_out)) || (kv_heads && (!k || !k_out)))
    return MRSA_ERR_INVALID_ARGUMENT;
  if (rotary_dim && table_rows && (!cos_table || !sin_table)) return MRSA_ERR_INVALID_ARGUMENT;
  RotaryArgs a = {};
  a.q = {q, q_batch_stride, q_row_stride, q_head_stride, q_out, seq_len * q_heads * head_dim,
         q_heads * head_dim, head_dim, (int)q_heads};
  a.k = {k, k_batch_stride, k_row_stride, k_head_stride, k_out, seq_len * kv_heads * head_dim,
         kv_heads * head_dim, head_dim, (int)kv_heads};
  a.cos_t = cos_table;
  a.sin_t = sin_table;
  a.table_rows = table_rows;
  a.positions = positions;
  a.ps_b = positions_batch_stride;
  a.ps_l = positions_row_stride;
  a.tokens = (int)(batch * seq_len);
  a.L = (int)seq_len;
  a.D = (int)head_dim;
  a.half = (int)(rotary_dim / 2);
  a.sign = inverse ? -1.f : 1.f;
  return dispatch<false>(a, dtype, interleaved, stream);
}

extern "C" int mrsa_paged_append_fwd(
    const void* q, int64_t q_batch_stride, int64_t q_row_stride, int64_t q_head_stride,
    const void* k, int64_t k_batch_stride, int64_t k_row_stride, int64_t k_head_stride,
    const void* v, int64_t v_batch_stride, int64_t v_row_stride, int64_t v_head_stride,
    const float* cos_table, const float* sin_table, int64_t table_rows, const int64_t* positions,
    int64_t positions_batch_stride, int64_t positions_row_stride, const int64_t* slots,
    int64_t slots_batch_stride, int64_t slots_row_stride, const int32_t* page_table,
    int64_t page_table_stride, int64_t table_pages, int64_t num_pages, int64_t page_size,
    void* k_pages, int64_t k_page_stride, int64_t k_slot_stride, int64_t k_pages_head_stride,
    void* v_pages, int64_t v_page_stride, int64_t v_slot_stride, int64_t v_pages_head_stride,
    int64_t batch, int64_t seq_len, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
    int64_t rotary_dim, int32_t dtype, int32_t interleaved, void* q_out, void* stream) {
  if (!sizes_ok(batch, seq_len, q_heads, kv_heads, head_dim, rotary_dim, table_rows) ||
      table_pages < 0 || num_pages < 0 || page_size <= 0)
    return MRSA_ERR_INVALID_ARGUMENT;
  if (dtype < MRSA_DTYPE_BF16 || dtype > MRSA_DTYPE_FP32) return MRSA_ERR_INVALID_ARGUMENT;
  if ((page_size & (page_size - 1)) != 0 || page_size > (1 << 20)) return MRSA_ERR_UNSUPPORTED;
  if (!sizes_fit(batch, seq_len, q_heads, kv_heads, head_dim) || table_pages > 0x7fffffff)
    return MRSA_ERR_UNSUPPORTED;
  if (batch * seq_len == 0 || q_heads + kv_heads == 0) return MRSA_OK;
  if ((q_heads && (!q || !q_out)) || !slots) return MRSA_ERR_INVALID_ARGUMENT;
  if (kv_heads && (!k || !v)) return MRSA_ERR_INVALID_ARGUMENT;
  // (the table is read for every row, also where there are no KV heads to place)
  if (table_pages && num_pages &&
      (!page_table || (kv_heads && (!k_pages || !v_pages || k_pages == v_pages))))
    return MRSA_ERR_INVALID_ARGUMENT;
  if (rotary_dim && table_rows && (!cos_table || !sin_table)) return MRSA_ERR_INVALID_ARGUMENT;
  RotaryArgs a = {};
  a.q = {q, q_batch_stride, q_row_stride, q_head_stride, q_out, seq_len * q_heads * head_dim,
         q_heads * head_dim, head_dim, (int)q_heads};
  a.k = {k, k_batch_stride, k_row_stride, k_head_stride,
         k_pages, k_page_stride, k_slot_stride, k_pages_head_stride, (int)kv_heads};
  a.v = {v, v_batch_stride, v_row_stride, v_head_stride,
         v_pages, v_page_stride, v_slot_stride, v_pages_head_stride, (int)kv_heads};
  a.cos_t = cos_table;
  a.sin_t = sin_table;
  a.table_rows = table_rows;
  a.positions = positions;
  a.ps_b = positions_batch_stride;
  a.ps_l = positions_row_stride;
  a.tokens = (int)(batch * seq_len);
  a.L = (int)seq_len;
  a.D = (int)head_dim;
  a.half = (int)(rotary_dim / 2);
  a.sign = 1.f;
  a.slots = slots;
  a.sl_b = slots_batch_stride;
  a.sl_l = slots_row_stride;
  a.table = page_table;
  a.table_stride = page_table_stride;
  a.table_width = num_pages ? (int)table_pages : 0;
  a.num_pages = num_pages;
  a.page_shift = __builtin_ctzll((uint64_t)page_size);
  return dispatch<true>(a, dtype, interleaved, stream);
}
