// Rows in 8-bit integers with one scale each: of activations as they are, of
// the root-mean-square norm of a residual sum, and of the gated activation;
// and the values that such rows stand for.
//
// A row y_0 .. y_{K-1} (fp32) with a = max |y_k| is held as
//     v_k = rint(y_k 127 / a)  in [-127, 127],   scale = a / 127,   y_k ~ v_k scale.
// a = 0: scale and values 0.  a not finite (an infinity or a NaN in the row):
// scale NaN and values 0, so that all that is made from the row is NaN.
//     quantize  y = x
//     norm      t = x + residual rounded to the tensors' type (and stored so),
//               y = t r w,  r = 1 / sqrt(mean t^2 + eps)
//     swiglu    y = g / (1 + exp(-g)) u
// No rounding between fp32 and the 8 bits.  r is the same for a whole row, so
// the values are those of t w, only the scale takes r, and one joint reduction
// gives sum t^2 and max |t w|.
#include "mrsa_device.h"

#include <type_traits>

using namespace mrsa;

namespace {

enum Op { kQuantize, kNorm, kAddNorm, kSwiglu };

// Element types.  Vector loads and stores of rows take addresses of any alignment (the hardware
// does; the packed type only keeps the compiler from assuming more).
struct Bf16 {
  typedef uint16_t elem;
  static __device__ __forceinline__ float widen(elem e) { return bf16_to_f32(e); }
  static __device__ __forceinline__ elem narrow(float f) { return (elem)f32_to_bf16(f); }
};
struct Fp16 {
  typedef uint16_t elem;
  static __device__ __forceinline__ float widen(elem e) {
    return (float)__builtin_bit_cast(_Float16, e);
  }
  static __device__ __forceinline__ elem narrow(float f) {
    return __builtin_bit_cast(elem, (_Float16)f);
  }
};
struct Fp32 {
  typedef float elem;
  static __device__ __forceinline__ float widen(elem e) { return e; }
  static __device__ __forceinline__ elem narrow(float f) { return f; }
};

template <class E, int N>
struct __attribute__((packed, aligned(1))) Pack {
  E e[N];
};

struct RowArgs {
  const void* x;         // swiglu: gate columns, then up columns
  const void* residual;  // norm, optional
  const void* weight;    // norm
  int64_t rows, K, x_stride, r_stride;  // in elements
  float eps;
  void* total;  // norm with residual: dense rows
  int8_t* values;
  float* scales;
};

// Eight elements from p on, or (SMALL: rows shorter than that) the K there are and zeros.
template <bool SMALL, class E>
__device__ __forceinline__ Pack<E, 8> load8(const E* p, int64_t K) {
  if constexpr (SMALL) {
    Pack<E, 8> w;
    for (int j = 0; j < 8; ++j) w.e[j] = j < K ? p[j] : E(0);
    return w;
  } else {
    return *reinterpret_cast<const Pack<E, 8>*>(p);
  }
}
template <class T, bool SMALL>
__device__ __forceinline__ void store8(typename T::elem* p, int64_t K, const float (&f)[8]) {
  typedef typename T::elem E;
  Pack<E, 8> w;
#pragma unroll
  for (int j = 0; j < 8; ++j) w.e[j] = T::narrow(f[j]);
  if constexpr (SMALL) {
    for (int j = 0; j < K; ++j) p[j] = w.e[j];
  } else {
    *reinterpret_cast<Pack<E, 8>*>(p) = w;
  }
}

// g / (1 + exp(-g)) for g from kFarGate on: the quotient by the hardware's reciprocal and one
// correction, which rounds it as a division does (the divisor, from 1 to 2^126, needs no scaling).
constexpr float kFarGate = -87.f;   // exp(87) is 0.71 2^126
__device__ __forceinline__ float silu(float g) {
  const float d = 1.f + expf(-g), r = rcp_hw(d);
  const float q = g * r;
  return fmaf(fmaf(-q, d, g), r, q);
}
// silu(g) up for g below kFarGate, where 1 + exp(-g) is exp(-g) but nears the end of fp32, whose
// reciprocal or quotient would lose it: the exponential in two halves around the other factor, so
// that nothing is lost before the product itself is (-inf: NaN, as -inf / inf).
__device__ __forceinline__ float far_gate(float g, float up) {
  const float h = expf(0.5f * g);
  return g * h * up * h;
}

// f + 1.5 2^23, whose low byte is the whole number nearest to f, ties to even.  (The product
// that f is stays a number of its own: an exact half, as bf16 rows have them, is a tie.)
__device__ __forceinline__ float whole(float f) {
#pragma clang fp contract(off)
  asm("" : "+v"(f));
  return f + 12582912.f;
}

constexpr uint32_t kInfBits = 0x7f800000u;
constexpr float kMostScale = 0x1.020406p121f;   // 127 times the next one passes fp32
constexpr uint32_t kFar = 0xffffffffu;   // above all magnitudes: the row has gates below kFarGate
__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
  v = max(v, (uint32_t)dpp_mov_i<0xb1>((int)v));   // quad_perm [1,0,3,2]
  v = max(v, (uint32_t)dpp_mov_i<0x4e>((int)v));   // quad_perm [2,3,0,1]
  v = max(v, (uint32_t)dpp_mov_i<0x141>((int)v));  // row_half_mirror
  v = max(v, (uint32_t)dpp_mov_i<0x140>((int)v));  // row_mirror
  auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max(r[0], r[1]);
}

// Sum and largest magnitude (as bits: a NaN's exceed infinity's) over the TPR threads of a row;
// every thread of the block takes part.
template <int TPR, bool SUM>
__device__ __forceinline__ void reduce(float& sum, uint32_t& top, float* red_sum,
                                       uint32_t* red_top) {
  if (SUM) sum = across4_sum(group16_sum(sum));
  top = wave_max_u(top);
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // (the words of an earlier reduction have been read)
    if ((threadIdx.x & 63) == 0) {
      if (SUM) red_sum[wave] = sum;
      red_top[wave] = top;
    }
    __syncthreads();
    sum = 0.f;
    top = 0;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) {
      if (SUM) sum += red_sum[i];
      top = max(top, red_top[i]);
    }
  }
}

// The same number; if AGAIN, one that the compiler keeps no addresses for ahead of its use.
template <bool AGAIN>
__device__ __forceinline__ int apart(int i) {
  if constexpr (AGAIN) asm volatile("" : "+v"(i));
  return i;
}

// TPR threads a row (a wave, so four rows a block; or the whole block), each with V units of
// eight elements; V = 0: rows of any length, read twice.  The last unit of a row ends with it and
// so may share elements with the one before: both write the same there, and the sum of squares
// takes them once.
//
// Bound by HBM where there are many rows, since a row stays in registers between its maximum and
// its values and so is read once (bf16, a large copy reaches 5.17 TB/s): 16384 rows of 3584
// quantized in 31 us (176 MB, 5.7 TB/s, partly from the caches), with the norm and the residual's
// sum in 77 us (411 MB, 5.3 TB/s); gated, of 18944, in 293 to 322 us (1552 MB, 4.8 to 5.3 TB/s),
// where the exponential, the quotient and the rounding, 30 vector instructions an element, keep
// the vector unit as busy as the memory.  One row of 3584 takes 2.9 us: a launch and three
// dependent steps (loads, reduction, stores).
template <class T, int OP, int TPR, int V, bool SMALL>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR,
                                  V == 5 && OP == kSwiglu && sizeof(typename T::elem) == 2 ? 6 : 1)
    int8_rows_kernel(RowArgs a) {
  typedef typename T::elem E;
  constexpr int THREADS = TPR < 256 ? 256 : TPR;
  constexpr int ROWS = THREADS / TPR;
  static_assert(TPR == 64 || ROWS == 1);
  constexpr int HELD = V > 0 ? V : 1;
  constexpr bool RES = OP == kAddNorm, NORM = OP == kNorm || RES;
  __shared__ float red_sum[THREADS / 64];
  __shared__ uint32_t red_top[THREADS / 64];
  const int sub = threadIdx.x % TPR;
  const int64_t units = (a.K + 7) / 8;
  auto start_of = [&](int64_t u) { return SMALL ? 0 : min(8 * u, a.K - 8); };
  for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < a.rows;
       row0 += (int64_t)gridDim.x * ROWS) {
    const bool there = row0 + threadIdx.x / TPR < a.rows;
    const int64_t row = there ? row0 + threadIdx.x / TPR : a.rows - 1;
    const E* const x = (const E*)a.x + row * a.x_stride;
    const E* const res = (const E*)a.residual + row * a.r_stride;
    const E* const w = (const E*)a.weight;
    float square = 0.f;   // norm: sum of (t down)^2
    float down = 1.f;     //       a power of two that keeps it in range
    uint32_t top_t = 0;   //       largest |t|
    uint32_t top = 0;     // largest magnitude of what `unit` gives
    float lowest = 0.f;   // swiglu: the least gate
    // What the unit at element s is made from: x or the gate, the residual or the other factor,
    // the weight.
    struct Unit {
      Pack<E, 8> x, other, w;
    };
    auto load = [&](int64_t s) {
      Unit n;
      n.x = load8<SMALL>(x + s, a.K);
      if constexpr (NORM) {
        n.w = load8<SMALL>(w + s, a.K);
        if constexpr (RES) n.other = load8<SMALL>(res + s, a.K);
      }
      if constexpr (OP == kSwiglu) n.other = load8<SMALL>(x + a.K + s, a.K);
      return n;
    };
    // Its values before the row's factor: x, t down w, or the product.
    auto unit = [&](const Unit& n, int64_t s, int repeated, bool first, auto far, float (&y)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = T::widen(n.x.e[j]);
      if constexpr (NORM) {
        if constexpr (RES) {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = T::widen(T::narrow(y[j] + T::widen(n.other.e[j])));
          if (first && there && repeated < 8)
            store8<T, SMALL>((E*)a.total + row * a.K + s, a.K, y);
        }
        float sq = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          top_t = max(top_t, magnitude(y[j]));
          y[j] *= down;
          sq = fmaf(y[j], y[j], sq);
        }
        if (repeated) {
          sq = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) sq = j < repeated ? sq : fmaf(y[j], y[j], sq);
        }
        square += sq;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] *= T::widen(n.w.e[j]);
      }
      if constexpr (OP == kSwiglu) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float g = y[j], up = T::widen(n.other.e[j]);
          if constexpr (far) {
            y[j] = g < kFarGate ? far_gate(g, up) : silu(g) * up;
          } else {
            lowest = fminf(lowest, g);
            y[j] = silu(g) * up;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, magnitude(y[j]));
    };
    float y[HELD][8];
    auto all_units = [&](bool first, auto far) {
      square = 0.f;
      top = top_t = 0;
      if constexpr (V > 0 && !far) {
        // (threads past the row take its last unit once more: no load depends on a branch)
        Unit n[HELD];
#pragma unroll
        for (int i = 0; i < V; ++i) n[i] = load(start_of(min<int64_t>(sub + i * TPR, units - 1)));
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int64_t u = sub + i * TPR, s = start_of(min(u, units - 1));
          unit(n[i], s, u < units ? (int)(8 * u - s) : 8, first, far, y[i]);
        }
      } else {
        for (int64_t u = apart<far>(sub); u < units; u += TPR) {
          const int64_t s = start_of(u);
          unit(load(s), s, (int)(8 * u - s), first, far, y[0]);
        }
      }
      if constexpr (OP == kSwiglu && !far) top = lowest < kFarGate ? kFar : top;
      reduce<TPR, NORM>(square, top, red_sum, red_top);
    };
    all_units(true, std::false_type{});
    float r = 1.f;
    bool far = false;
    if constexpr (OP == kSwiglu) {
      // Again, with the form for gates that far down, and unit by unit, so that the other rows
      // keep the registers that they had (80 for 18944 values of 16 bits: three blocks a CU, 290
      // us instead of 314).  A test of each unit in its place slows them more (3584 values: 64 us
      // instead of 59); all rows of 18944 taken again are 620.
      far = top == kFar;
      if (far) all_units(false, std::true_type{});
    }
    if constexpr (NORM) {
      // t^2 or t w past fp32 (|t| above 1.8e19, or above 1 beside a large weight): again with t
      // times a power of two that takes the largest |t| to between 1/4 and 1/2, so that t w is
      // finite.  A row that holds an infinity or a NaN comes here, too, and stays what it is.
      const bool past = !(square < __uint_as_float(kInfBits)) || top >= kInfBits;
      if (__any(past)) {  // (the same in every wave of a row)
        float none = 0.f;
        reduce<TPR, false>(none, top_t, red_sum, red_top);
        const int e = past ? (int)(top_t >> 23) - 127 : -2;
        down = ldexpf(1.f, -2 - min(e, 127));
        all_units(false, std::false_type{});
      }
      r = rsqrtf(square / (float)a.K + a.eps * down * down);
    }
    const float most = __uint_as_float(top);
    // (the norm's y may pass fp32 where t w does not)
    const bool bad = top >= kInfBits || (NORM && !(most * r < __uint_as_float(kInfBits)));
    // (rows below 2^-100, whose 127 / a could pass fp32, are lifted first)
    const float lift = most < 0x1p-100f ? 0x1p100f : 1.f;
    const float up = bad || top == 0 ? 0.f : 1.f / (most * lift) * 127.f;
    auto put = [&](int64_t s, float (&f)[8]) {
      uint32_t v[2];
      if (lift != 1.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= lift;
      }
      // |f up| <= 127 (1 + 2^-22), so the whole number is at most 127.
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = __float_as_uint(whole(f[4 * h + j] * up));
        const uint32_t lo = __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(q[3], q[2], 0x04000c0cu);
        v[h] = bad ? 0u : lo | hi;
      }
      int8_t* const to = a.values + row * a.K + s;
      if constexpr (SMALL) {
        for (int j = 0; j < a.K; ++j) to[j] = (int8_t)(v[j >> 2] >> (8 * (j & 3)));
      } else {
        *reinterpret_cast<Pack<uint32_t, 2>*>(to) = Pack<uint32_t, 2>{{v[0], v[1]}};
      }
    };
    if (there) {
      auto read_again = [&](auto far) {
        for (int64_t u = apart<far>(sub); u < units; u += TPR) {
          const int64_t s = start_of(u);
          unit(load(s), s, 0, false, far, y[0]);
          put(s, y[0]);
        }
      };
      if (OP == kSwiglu && far) {
        read_again(std::true_type{});
      } else if constexpr (V > 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int64_t u = sub + i * TPR;
          if (u < units) put(start_of(u), y[i]);
        }
      } else {
        read_again(std::false_type{});
      }
      if (sub == 0) a.scales[row] = bad ? __builtin_nanf("") : fminf(most * r / 127.f, kMostScale);
    }
  }
}

// Values times their row's scale: a block covers 16 columns a thread (x) of rows (y).  Bound by
// HBM: 16384 rows of 3584 to bf16 27 us (6.5 TB/s, the values partly from the caches), of 18944
// 189 us (4.9 TB/s).
template <class T, bool SMALL>
__global__ void __launch_bounds__(256)
    int8_back_kernel(const int8_t* __restrict__ values, int64_t stride,
                     const float* __restrict__ scales, int64_t rows, int64_t K,
                     typename T::elem* __restrict__ out) {
  typedef typename T::elem E;
  const int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (u >= (K + 15) / 16) return;
  const int64_t s = SMALL ? 0 : min(16 * u, K - 16);
  for (int64_t row = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; row < rows;
       row += (int64_t)gridDim.y * blockDim.y) {
    const int8_t* const p = values + row * stride + s;
    E* const to = out + row * K + s;
    const float scale = scales[row];
    if constexpr (SMALL) {
      for (int j = 0; j < K; ++j) to[j] = T::narrow((float)p[j] * scale);
    } else {
      const Pack<uint32_t, 4> v = *reinterpret_cast<const Pack<uint32_t, 4>*>(p);
      Pack<E, 16> o;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        o.e[j] = T::narrow((float)(int8_t)(v.e[j >> 2] >> (8 * (j & 3))) * scale);
      *reinterpret_cast<Pack<E, 16>*>(to) = o;
    }
  }
}

template <class T, int OP, int TPR, int V, bool SMALL = false>
void launch_rows(const RowArgs& a, hipStream_t stream) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR;
  const int64_t blocks = (a.rows + THREADS / TPR - 1) / (THREADS / TPR);
  hipLaunchKernelGGL((int8_rows_kernel<T, OP, TPR, V, SMALL>),
                     dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(THREADS), 0, stream,
                     a);
}

// A wave a row up to 1024 elements (no barriers: 16384 rows of 1024 9.6 us, by blocks of 256
// 13.3), then a block whose threads hold the row in registers, with as few units a thread as
// leaves no thread idle: us, bf16,
//             rows    elements   256 threads (units)   512           1024
//   quantize  16384       3584   27.4 (2)              31.4 (1)      55.3 (1)
//   norm      16384       3584   70.5 (2)              74.7 (1)      103 (1)
//   swiglu       32       3584   3.0 (2)               2.8 (1)
//   swiglu    16384       3584   51.8 (2)              59.2 (1)      101 (1)
//   swiglu    16384       8192   128 (4)               118 (2)       122 (1)
//   norm      16384      12288   276 (8)               242 (3)       291 (2)
//   swiglu    16384      18944   297 (10)              284 (5)       309 (3)
//   norm      16384      18944   549 (10)              446 (5)       434 (3)
// (Gated rows of 2049 to 4096 elements take 512 threads for the few rows of a decode block, and in
// fp32 also for many: 16384 rows of 3584 94 us, 256 threads 98.)  Past 20480 elements the row is
// read twice, by 1024 threads (8192 rows of 32768: quantize 176 us, 512 threads 192; one row of
// them 3.8 and 5.0).
template <class T, int OP>
void rows_of(const RowArgs& a, hipStream_t stream) {
  const int64_t units = (a.K + 7) / 8;
  if (a.K < 8) launch_rows<T, OP, 64, 1, true>(a, stream);
  else if (units <= 64) launch_rows<T, OP, 64, 1>(a, stream);
  else if (units <= 128) launch_rows<T, OP, 64, 2>(a, stream);
  else if (units <= 256) launch_rows<T, OP, 256, 1>(a, stream);
  else if (units <= 512 && OP == kSwiglu) launch_rows<T, OP, 512, 1>(a, stream);
  else if (units <= 512) launch_rows<T, OP, 256, 2>(a, stream);
  else if (units <= 1024) launch_rows<T, OP, 512, 2>(a, stream);
  else if (units <= 1536) launch_rows<T, OP, 512, 3>(a, stream);
  else if (units <= 2560) launch_rows<T, OP, 512, 5>(a, stream);
  else launch_rows<T, OP, 1024, 0>(a, stream);
}

template <int OP>
int rows_of_dtype(const RowArgs& a, int32_t dtype, hipStream_t stream) {
  switch (dtype) {
    case MRSA_DTYPE_BF16: rows_of<Bf16, OP>(a, stream); break;
    case MRSA_DTYPE_FP16: rows_of<Fp16, OP>(a, stream); break;
    case MRSA_DTYPE_FP32: rows_of<Fp32, OP>(a, stream); break;
    default: return MRSA_ERR_UNSUPPORTED;
  }
  return mrsa_launch_status();
}

bool misaligned(const void* p, int32_t dtype) {
  return (uintptr_t)p % (dtype == MRSA_DTYPE_FP32 ? 4 : 2) != 0;
}
bool known_dtype(int32_t dtype) {
  return dtype == MRSA_DTYPE_BF16 || dtype == MRSA_DTYPE_FP16 || dtype == MRSA_DTYPE_FP32;
}
// Sizes whose addresses could pass 63 bits.
bool too_large(int64_t rows, int64_t K, int64_t stride) {
  return K > ((int64_t)1 << 31) || rows > ((int64_t)1 << 40) ||
         rows > ((int64_t)1 << 56) / std::max<int64_t>(1, std::max(K, stride));
}

template <class T>
void back(const int8_t* values, int64_t stride, const float* scales, int64_t rows, int64_t K,
          void* out, hipStream_t stream) {
  const int64_t units = (K + 15) / 16;
  unsigned tx = 1;
  while (tx < 256 && tx < units) tx *= 2;
  const unsigned ty = 256 / tx;
  // (four rows a thread keep the number of blocks low where there are many)
  const int64_t by =
      std::min<int64_t>((rows + ty - 1) / ty, std::max<int64_t>(2048, rows / ty / 4));
  const dim3 grid((unsigned)((units + tx - 1) / tx), (unsigned)std::min<int64_t>(by, 65535));
  auto kern = K < 16 ? int8_back_kernel<T, true> : int8_back_kernel<T, false>;
  hipLaunchKernelGGL(kern, grid, dim3(tx, ty), 0, stream, values, stride, scales, rows, K,
                     (typename T::elem*)out);
}

}  // namespace

extern "C" int mrsa_quantize_rows_fwd(const void* x, int64_t x_row_stride, int64_t rows,
                                      int64_t dim, int32_t dtype, int8_t* values, float* scales,
                                      void* stream) {
  if (rows < 0 || dim < 0 || x_row_stride < 0) return MRSA_ERR_INVALID_ARGUMENT;
  if (!known_dtype(dtype) || dim == 0 || too_large(rows, dim, x_row_stride))
    return MRSA_ERR_UNSUPPORTED;
  if (rows == 0) return MRSA_OK;
  if (!x || !values || !scales || misaligned(x, dtype) || (uintptr_t)scales % 4 != 0)
    return MRSA_ERR_INVALID_ARGUMENT;
  RowArgs a = {x, nullptr, nullptr, rows, dim, x_row_stride, 0, 0.f, nullptr, values, scales};
  return rows_of_dtype<kQuantize>(a, dtype, (hipStream_t)stream);
}

extern "C" int mrsa_add_rms_norm_int8_fwd(const void* x, int64_t x_row_stride,
                                          const void* residual, int64_t residual_row_stride,
                                          const void* weight, int64_t rows, int64_t dim, float eps,
                                          int32_t dtype, void* total, int8_t* values,
                                          float* scales, void* stream) {
  if (rows < 0 || dim < 0 || x_row_stride < 0 || residual_row_stride < 0 || !(eps >= 1e-24f) ||
      !(eps <= 1e24f))
    return MRSA_ERR_INVALID_ARGUMENT;
  if (!known_dtype(dtype) || dim == 0 || too_large(rows, dim, x_row_stride) ||
      too_large(rows, dim, residual_row_stride))
    return MRSA_ERR_UNSUPPORTED;
  if (rows == 0) return MRSA_OK;
  if (!x || !weight || !values || !scales || !residual != !total || misaligned(x, dtype) ||
      misaligned(residual, dtype) || misaligned(weight, dtype) || misaligned(total, dtype) ||
      (uintptr_t)scales % 4 != 0)
    return MRSA_ERR_INVALID_ARGUMENT;
  RowArgs a = {x,   residual, weight, rows, dim, x_row_stride, residual_row_stride,
               eps, total,    values, scales};
  return residual ? rows_of_dtype<kAddNorm>(a, dtype, (hipStream_t)stream)
                  : rows_of_dtype<kNorm>(a, dtype, (hipStream_t)stream);
}

extern "C" int mrsa_swiglu_int8_fwd(const void* gate_up, int64_t row_stride, int64_t rows,
                                    int64_t dim, int32_t dtype, int8_t* values, float* scales,
                                    void* stream) {
  if (rows < 0 || dim < 0 || row_stride < 0) return MRSA_ERR_INVALID_ARGUMENT;
  if (!known_dtype(dtype) || dim == 0 || dim > (int64_t)1 << 30 ||
      too_large(rows, 2 * dim, row_stride))
    return MRSA_ERR_UNSUPPORTED;
  if (rows == 0) return MRSA_OK;
  if (!gate_up || !values || !scales || misaligned(gate_up, dtype) || (uintptr_t)scales % 4 != 0)
    return MRSA_ERR_INVALID_ARGUMENT;
  RowArgs a = {gate_up, nullptr, nullptr, rows, dim, row_stride, 0, 0.f, nullptr, values, scales};
  return rows_of_dtype<kSwiglu>(a, dtype, (hipStream_t)stream);
}

extern "C" int mrsa_dequantize_rows_fwd(const int8_t* values, int64_t row_stride,
                                        const float* scales, int64_t rows, int64_t dim,
                                        int32_t dtype, void* out, void* stream) {
  if (rows < 0 || dim < 0 || row_stride < 0) return MRSA_ERR_INVALID_ARGUMENT;
  if (!known_dtype(dtype) || too_large(rows, dim, row_stride)) return MRSA_ERR_UNSUPPORTED;
  if (rows == 0 || dim == 0) return MRSA_OK;
  if (!values || !scales || !out || misaligned(out, dtype) || (uintptr_t)scales % 4 != 0)
    return MRSA_ERR_INVALID_ARGUMENT;
  switch (dtype) {
    case MRSA_DTYPE_BF16: back<Bf16>(values, row_stride, scales, rows, dim, out,
                                     (hipStream_t)stream); break;
    case MRSA_DTYPE_FP16: back<Fp16>(values, row_stride, scales, rows, dim, out,
                                     (hipStream_t)stream); break;
    default: back<Fp32>(values, row_stride, scales, rows, dim, out, (hipStream_t)stream);
  }
  return mrsa_launch_status();
}
