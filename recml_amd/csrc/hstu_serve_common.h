// What the sources of libhstu_serve.so share: the error text, bf16 conversions, the cache's geometry.

#ifndef HSTU_SERVE_COMMON_H_
#define HSTU_SERVE_COMMON_H_

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "hstu_serve.h"

// Stores the message that hstu_serve_last_error() returns on this thread; returns `code`.
__attribute__((visibility("hidden"))) int serve_fail(int code, const char* fmt, ...);
__attribute__((visibility("hidden"))) void serve_clear_error();
// Whether the pages are ones that the kernels take.
__attribute__((visibility("hidden"))) int serve_check_pages(const HstuKvPages& pages);
// The status of the launch just made.
__attribute__((visibility("hidden"))) int serve_launched(const char* what);

namespace {

typedef __bf16 bf16_t;
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;

constexpr int64_t SERVE_THREADS = 0xffffffffll;      // of one launch: a dimension's threads are counted in 32 bits

inline bool serve_aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  floatx2 f = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __builtin_bit_cast(float, w[i] << 16);
    f[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
  }
}

// 2^(e - 127) for an exponent byte in [1, 254]
__device__ __forceinline__ float power_of(uint32_t e) { return __builtin_bit_cast(float, e << 23); }

// The row of sequence b's event at `place`, as an index over all pages' rows of one head 0: page * H * page_size + slot;
// -1 where the cache does not hold it.
__device__ __forceinline__ int64_t kv_row(const HstuKvPages& p, int b, int64_t place) {
  if (place < 0 || place >= (int64_t)p.table_pages * p.page_size) return -1;
  const int at = (int)(place / p.page_size);
  const int page = p.page_table[(int64_t)b * p.table_pages + at];
  if (page < 0 || page >= p.n_pages) return -1;
  return (int64_t)page * p.H * p.page_size + (place - (int64_t)at * p.page_size);
}

}  // namespace

#endif  // HSTU_SERVE_COMMON_H_
