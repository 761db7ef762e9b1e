// What the sources of libhstu_rows8.so share: the error text, conversions, the geometry of rows in 8 bits.

#ifndef HSTU_ROWS8_COMMON_H_
#define HSTU_ROWS8_COMMON_H_

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "hstu_rows8.h"

// Stores the message that hstu_rows8_last_error() returns on this thread; returns `code`.
__attribute__((visibility("hidden"))) int rows8_fail(int code, const char* fmt, ...);
__attribute__((visibility("hidden"))) void rows8_clear_error();
// Whether they are rows that the kernels take.
__attribute__((visibility("hidden"))) int rows8_check(const HstuRows8& rows, const char* name);
// The status of the launch just made.
__attribute__((visibility("hidden"))) int rows8_launched(const char* what);

namespace {

typedef __bf16 bf16_t;
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int BLOCK = 128;                           // values that share an exponent
constexpr int64_t ROWS8_THREADS = 0xffffffffll;      // of one launch: a dimension's threads are counted in 32 bits

__host__ __device__ inline int rows8_blocks(int width) { return (width + BLOCK - 1) / BLOCK; }
inline bool rows8_aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  floatx2 f = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}

__device__ __forceinline__ void unpack8(const uint4v& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __builtin_bit_cast(float, v[i] << 16);
    f[2 * i + 1] = __builtin_bit_cast(float, v[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4v pack8(const float (&y)[8]) {
  return uint4v{pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7])};
}

// 2^(e - 127) for an exponent byte in [1, 254]
__device__ __forceinline__ float power_of(uint32_t e) { return __builtin_bit_cast(float, e << 23); }

}  // namespace

#endif  // HSTU_ROWS8_COMMON_H_
