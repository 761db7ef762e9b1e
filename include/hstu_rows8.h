/* C ABI of libhstu_rows8.so: a block's steps (recml/layers/keras/hstu.py:442-474) on rows kept in 8 bits, for inference on gfx950.
 *
 *   hstu_rows8_norm   rows, normed or as they are, into 8 bits: what stands in front of a product (the block's input norm,
 *                     hstu.py:442; its attention norm with the U gate, hstu.py:471-472), the residual's addition with it
 *   hstu_rows8_read   the values that such rows stand for
 *   hstu_rows8_gemm   the product of two of them (hstu.py:444-449, 473-474), with bias, residual and SiLU behind it
 *
 * The format: a row is its codes, e4m3, in 128 ceil(width / 128) bytes, and one exponent byte for each block of 128 of them.  A block
 * stands for its codes times 2^(e - 127) of its exponent byte e, the smallest in [1, 246] under which the block's largest magnitude rounds
 * to a code (at most 464 times the power; no code stands for more than fp32 holds), so every value is off by at most half of its step;
 * values round to the nearest code, ties to the even one, past the largest to the largest.  A block that holds a value which is not finite
 * has codes of zero and an exponent of 255: it stands for NaN.  Codes past the width are zeros.
 *   codes      [rows, 128 ceil(width / 128)]
 *   exponents  [ceil(width / 512), rows, 4]: those of four blocks of a row side by side (1 where there is no block)
 * The powers are what the scaled matrix instructions take, so a product needs no multiplication by scales of its own.
 *
 * Plain pointers and sizes: no framework types.  Every function returns 0 or a negative HstuRows8Status; the message of the last failure
 * on the calling thread is at hstu_rows8_last_error().  Work is enqueued on `stream` on the current device; nothing is allocated.
 */
#ifndef HSTU_ROWS8_H_
#define HSTU_ROWS8_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HSTU_ROWS8_ABI_VERSION 1

typedef enum HstuRows8Status {
  HSTU_ROWS8_OK = 0,
  HSTU_ROWS8_ERR_NULL = -1,
  HSTU_ROWS8_ERR_VERSION = -2,
  HSTU_ROWS8_ERR_SHAPE = -4,
  HSTU_ROWS8_ERR_LAUNCH = -6
} HstuRows8Status;

typedef enum HstuRows8Dtype { HSTU_ROWS8_BF16 = 0, HSTU_ROWS8_FP32 = 1 } HstuRows8Dtype;
typedef enum HstuRows8NormKind { HSTU_ROWS8_AS_IS = 0, HSTU_ROWS8_LAYER = 1, HSTU_ROWS8_RMS = 2 } HstuRows8NormKind;

/* Rows in 8 bits.  codes on a 16-byte boundary, exponents on a 4-byte one; width from 1 to HSTU_ROWS8_MAX_WIDTH, rows up to 2^31 - 1. */
#define HSTU_ROWS8_MAX_WIDTH 32768
typedef struct HstuRows8 {
  void* codes;
  void* exponents;
  int64_t rows;
  int32_t width, reserved0;
} HstuRows8;

/* s = x (+ add, rounded to their type: it is stored at `sum` if that is given, and the norm is of the rounded rows)
 *   HSTU_ROWS8_LAYER  y = (s - mean) * rstd * gamma + beta   mean and (biased) variance of the row, rstd = 1 / sqrt(variance + eps)
 *   HSTU_ROWS8_RMS    y = s * rstd * gamma + beta            rstd = 1 / sqrt(mean of s^2 + eps)
 *   HSTU_ROWS8_AS_IS  y = x, with nothing added and no gate
 * rows = (gate *) y in 8 bits.  Statistics and products in fp32, or in 64 bits for rows in fp32, and one rounding to the codes.  A sum of squares
 * past fp32's largest (for rows in fp32: a mean of squares) counts as infinite: rstd = 0.  Rows in bf16 whose variance (mean of s^2) + eps lies
 * below 2^-126 have no rstd and stand for NaN: only an eps that small lets them.  x, add, gate,
 * sum: [rows, width] of `dtype` with row strides in elements (any alignment of the type); add and gate may be null, sum with add; sum may be
 * x or add (with its stride), otherwise no output may overlap an input.  gamma [width] of `dtype` (a norm needs it), beta likewise or null. */
typedef struct HstuRows8NormArgs {
  uint32_t struct_size;   /* sizeof(HstuRows8NormArgs) */
  uint32_t version;       /* HSTU_ROWS8_ABI_VERSION    */
  HstuRows8 rows;
  int32_t norm, dtype;
  float eps;
  int32_t reserved0;
  const void* x;
  const void* add;
  const void* gate;
  void* sum;
  int64_t x_stride, add_stride, gate_stride, sum_stride;
  const void* gamma;
  const void* beta;
} HstuRows8NormArgs;

int hstu_rows8_norm(const HstuRows8NormArgs* args, void* stream);

/* out [rows, width] of `dtype` (exact in fp32; in bf16 down to its smallest values), row stride in elements. */
typedef struct HstuRows8ReadArgs {
  uint32_t struct_size;   /* sizeof(HstuRows8ReadArgs) */
  uint32_t version;       /* HSTU_ROWS8_ABI_VERSION    */
  HstuRows8 rows;
  void* out;
  int64_t out_stride;
  int32_t dtype, reserved0;
} HstuRows8ReadArgs;

int hstu_rows8_read(const HstuRows8ReadArgs* args, void* stream);

/* out[m, n] = act(sum_k x[m, k] w[n, k] + c[m, n] + bias[n]), x and w the values that their rows stand for, of one width; sums in fp32,
 * one rounding to `dtype`.  For bf16 results each product is cut to 2^-13 of the largest of its eight neighbours along k before it is
 * added (what the matrix instructions on codes do); for fp32 results every product is exact, but that blocks under the smallest two exponents
 * count with their values to the nearest multiple of 2^-133 (bf16's least, as which codes are multiplied there).  out and c: [x.rows, w.rows] of `dtype` with row
 * strides in elements, bias [w.rows]; c and bias may be null; c may be out (with its stride).  Any alignment of the type; pointers and
 * strides of whole 16 bytes, and as many columns, run faster.  activation: 1 = silu, 0 = none. */
typedef struct HstuRows8GemmArgs {
  uint32_t struct_size;   /* sizeof(HstuRows8GemmArgs) */
  uint32_t version;       /* HSTU_ROWS8_ABI_VERSION    */
  HstuRows8 x;
  HstuRows8 w;
  int32_t dtype, activation;
  void* out;
  const void* c;
  const void* bias;
  int64_t out_stride, c_stride;
} HstuRows8GemmArgs;

int hstu_rows8_gemm(const HstuRows8GemmArgs* args, void* stream);

int hstu_rows8_abi_version(void);
const char* hstu_rows8_last_error(void);

#ifdef __cplusplus
}
#endif

#endif  /* HSTU_ROWS8_H_ */
