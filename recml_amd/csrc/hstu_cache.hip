// The pages of a cache of keys and values in 4 or 8 bits, for gfx950 (MI355X): see include/hstu_serve.h.
//
//   hstu_kv_write   rows of new events -> codes and block exponents
//   hstu_kv_read    codes and exponents -> rows
//
// Both are passes over memory.  One workgroup takes 32 places of one (sequence, head), keys and values: page sizes are multiples of 32 and
// the places start at a multiple of 32, so it stays inside one page, its codes are one run of 32 rows and its exponents one
// run of 32 bytes per block.

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "hstu_serve_common.h"

namespace {
thread_local char g_err[512] = "";
}

int serve_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

void serve_clear_error() { g_err[0] = 0; }

int serve_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HSTU_SERVE_OK : serve_fail(HSTU_SERVE_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

namespace {

constexpr int TILE = 32;     // places of one workgroup

typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

// One of the two tensors of a call.
struct Side {
  uint8_t* codes;
  uint8_t* scales;
  void* rows;
  int64_t sb, st, sh;
};

struct Params {
  HstuKvPages g;
  Side side[2];
  const int32_t* starts;
  const int32_t* offsets;
  int64_t total;
  int32_t per_seq, tiles;
};

// The rows of sequence b that are there: the first one's index and their number.
__device__ __forceinline__ void rows_of(const Params& p, int b, int64_t* first, int* count) {
  if (!p.offsets) { *first = 0; *count = p.per_seq; return; }
  int64_t o0 = p.offsets[b], o1 = p.offsets[b + 1];
  o0 = o0 < 0 ? 0 : o0 > p.total ? p.total : o0;
  o1 = o1 < o0 ? o0 : o1 > p.total ? p.total : o1;
  *first = o0;
  *count = (int)(o1 - o0 < p.per_seq ? o1 - o0 : p.per_seq);
}

// Eight values of a row as they lie in memory.
template <bool F32>
struct Eight { uint4 w[F32 ? 2 : 1]; };

template <bool F32>
__device__ __forceinline__ void load8(const void* base, int64_t at, Eight<F32>& x) {
  const uint4v* const from = (const uint4v*)((const char*)base + at * (F32 ? 4 : 2));
  // (rows are read once.  Past the caches where a wave's loads are whole lines: 131 k rows of 8 x 128 in bf16 136 us without, 124
  // with; fp32, two loads a lane: 118 without, 127 with)
  if constexpr (F32) {
    x.w[0] = __builtin_bit_cast(uint4, from[0]);
    x.w[1] = __builtin_bit_cast(uint4, from[1]);
  } else {
    x.w[0] = __builtin_bit_cast(uint4, __builtin_nontemporal_load(from));
  }
}

// The largest of the eight magnitudes, as fp32 bits (0x7f800000 and more: an infinity, a NaN).
template <bool F32>
__device__ __forceinline__ uint32_t largest(const Eight<F32>& x) {
  if constexpr (F32) {
    const uint32_t w[8] = {x.w[0].x, x.w[0].y, x.w[0].z, x.w[0].w, x.w[1].x, x.w[1].y, x.w[1].z, x.w[1].w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = (w[i] & 0x7fffffffu) > m ? w[i] & 0x7fffffffu : m;
    return m;
  } else {
    const uint32_t w[4] = {x.w[0].x, x.w[0].y, x.w[0].z, x.w[0].w};
    ushort2v m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(ushort2v, w[i] & 0x7fff7fffu));
    return (uint32_t)(m[0] > m[1] ? m[0] : m[1]) << 16;
  }
}

// Their codes under the power 2^(e - 127).
template <int BITS, bool F32>
__device__ __forceinline__ uint2 codes_of(const Eight<F32>& x, uint32_t e) {
  uint32_t code[2] = {0, 0};
  if constexpr (BITS == 4) {
    // the hardware's scaled conversion: to the nearest code, ties to the even one, past the largest to the largest
    const float power = power_of(e);
    if constexpr (F32) {
      const float* const y = (const float*)&x;
      uint32_t c = 0;
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[0], y[1], power, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2], y[3], power, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[4], y[5], power, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[6], y[7], power, 3);
      code[0] = c;
    } else {
      uint32_t c = 0;
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, x.w[0].x), power, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, x.w[0].y), power, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, x.w[0].z), power, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, x.w[0].w), power, 3);
      code[0] = c;
    }
  } else {
    float y[8];
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = ((const float*)&x)[i];
    } else {
      unpack8(x.w[0], y);
    }
    const float inverse = power_of(254 - e);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __builtin_amdgcn_fmed3f(y[i] * inverse, -448.f, 448.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
      code[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], c, true);
    }
  }
  return uint2{code[0], code[1]};
}

constexpr int threads_of(int lpr) { return lpr < 8 ? TILE * lpr : 256; }

// What a workgroup's 32 places are: the rows of one (sequence, head) from place `base` on.
struct Tile {
  int64_t t0;            // the sequence's row at the tile's first place (may be negative)
  int64_t first;         // the sequence's first row
  int count;             // and how many it has
  int h, b;
  int64_t row0;          // kv_row of the tile's first place
};

__device__ __forceinline__ bool tile_of(const Params& p, Tile* t) {
  t->h = blockIdx.x % p.g.H;
  const int tile = blockIdx.x / p.g.H % p.tiles;
  t->b = blockIdx.x / p.g.H / p.tiles;
  rows_of(p, t->b, &t->first, &t->count);
  const int64_t start = p.starts[t->b];
  // (the first tile's first place: the multiple of 32 at or below `start`, which may be negative)
  const int64_t base = (start - (((start % TILE) + TILE) % TILE)) + (int64_t)tile * TILE;
  t->t0 = base - start;
  if (t->t0 >= t->count) return false;
  t->row0 = kv_row(p.g, t->b, base);
  return true;
}

// LPR lanes per row (8 values each); all of a thread's rows, of the keys and of the values, are on their way before the first is
// worked on: 65.5 k rows of 8 x 128, 340 MB in and out, 128 us with one load at a time, 64 so (5.3 TB/s, past a large copy's rate).
template <int BITS, bool F32, int LPR>
__global__ __launch_bounds__(threads_of(LPR)) void hstu_kv_write_kernel(const Params p) {
  constexpr int ROWS = threads_of(LPR) / LPR, PASSES = TILE / ROWS;
  Tile t;
  if (!tile_of(p, &t) || t.row0 < 0) return;
  const int d = p.g.d, page = p.g.page_size, lane = threadIdx.x % LPR, r0 = threadIdx.x / LPR;
  const int blocks = (d + 31) / 32, row_bytes = d * BITS / 8;
  Eight<F32> x[2][PASSES];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int n = 0; n < PASSES; ++n) {
      const int64_t row = t.t0 + r0 + n * ROWS;
      x[s][n] = Eight<F32>{};
      if (row >= 0 && row < t.count && lane * 8 < d)
        load8<F32>(p.side[s].rows, (p.offsets ? 0 : (int64_t)t.b * p.side[s].sb) + (t.first + row) * p.side[s].st + (int64_t)t.h * p.side[s].sh + lane * 8, x[s][n]);
    }
  const int64_t head0 = t.row0 + (int64_t)t.h * page;               // row of the tile's first place in its head's rows
  const int64_t page_head = t.row0 / page + t.h, slot0 = t.row0 % page;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int n = 0; n < PASSES; ++n) {
      const int r = r0 + n * ROWS;
      const int64_t row = t.t0 + r;
      // a block's four lanes, then the row's
      uint32_t top = largest<F32>(x[s][n]);
#pragma unroll
      for (int m = 1; m < 4; m <<= 1) {
        const uint32_t o = __shfl_xor(top, m, 64);
        top = o > top ? o : top;
      }
      uint32_t bad = top >= 0x7f800000u;
#pragma unroll
      for (int m = 4; m < LPR; m <<= 1) bad |= __shfl_xor(bad, m, 64);
      // the exponent: floor(log2 top) less the largest code's, one more where top is past the middle above that code
      constexpr int TOP_EXP = BITS == 4 ? 2 : 8;
      constexpr uint32_t PAST = BITS == 4 ? 0x600000u : 0x680000u;      // mantissas of 1.75 and 1.8125
      constexpr int MOST = BITS == 4 ? 252 : 246;                       // (no code stands for more than fp32 holds: such rows saturate)
      int e = (int)(top >> 23) - TOP_EXP + ((top & 0x7fffffu) > PAST ? 1 : 0);
      e = e < 1 ? 1 : e > MOST ? MOST : e;                              // (top = 0 too)
      const uint2 code = codes_of<BITS, F32>(x[s][n], (uint32_t)e);
      if (row < 0 || row >= t.count || lane * 8 >= d) continue;
      uint8_t* const to = p.side[s].codes + (head0 + r) * row_bytes + lane * BITS;
      if constexpr (BITS == 4) *(uint32_t*)to = bad ? 0 : code.x;
      else *(uint2*)to = bad ? uint2{0, 0} : code;
      if (lane % 4 == 0) p.side[s].scales[(page_head * blocks + lane / 4) * page + slot0 + r] = (uint8_t)(bad ? 255 : e);
    }
}

// The same tiles the other way: 65.5 k rows of 8 x 128 from 4 bits, 340 MB, in 49 us: its stores are most of them.
template <int BITS, bool F32, int LPR>
__global__ __launch_bounds__(threads_of(LPR)) void hstu_kv_read_kernel(const Params p) {
  constexpr int ROWS = threads_of(LPR) / LPR, PASSES = TILE / ROWS;
  Tile t;
  if (!tile_of(p, &t)) return;
  const int d = p.g.d, page = p.g.page_size, lane = threadIdx.x % LPR, r0 = threadIdx.x / LPR;
  if (lane * 8 >= d) return;
  const int blocks = (d + 31) / 32, row_bytes = d * BITS / 8;
  const int64_t head0 = t.row0 + (int64_t)t.h * page, page_head = t.row0 / page + t.h, slot0 = t.row0 % page;
  uint2 code[2][PASSES];
  uint32_t e[2][PASSES];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int n = 0; n < PASSES; ++n) {
      const int r = r0 + n * ROWS;
      const int64_t row = t.t0 + r;
      code[s][n] = uint2{0, 0};
      e[s][n] = 1;
      if (t.row0 < 0 || row < 0 || row >= t.count) continue;
      const uint8_t* const from = p.side[s].codes + (head0 + r) * row_bytes + lane * BITS;
      if constexpr (BITS == 4) code[s][n].x = *(const uint32_t*)from;
      else code[s][n] = *(const uint2*)from;
      e[s][n] = p.side[s].scales[(page_head * blocks + lane / 4) * page + slot0 + r];
    }
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int n = 0; n < PASSES; ++n) {
      const int64_t row = t.t0 + r0 + n * ROWS;
      if (row < 0 || row >= t.count) continue;
      const float power = e[s][n] == 255u ? __builtin_nanf("") : power_of(e[s][n]);
      const uint2 w = code[s][n];
      floatx2 y[4];
      if constexpr (BITS == 4) {
        y[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.0f, 0); y[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.0f, 1);
        y[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.0f, 2); y[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w.x, 1.0f, 3);
      } else {
        y[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false); y[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true);
        y[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false); y[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
      }
      // (a product in fp32: exact, and a NaN for a row that is not finite, zeros included)
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = floatx2{y[i][0] * power, y[i][1] * power};
      const int64_t at = (p.offsets ? 0 : (int64_t)t.b * p.side[s].sb) + (t.first + row) * p.side[s].st + (int64_t)t.h * p.side[s].sh + lane * 8;
      if constexpr (F32) {
        floatx4* const to = (floatx4*)((float*)p.side[s].rows + at);
        to[0] = floatx4{y[0][0], y[0][1], y[1][0], y[1][1]};
        to[1] = floatx4{y[2][0], y[2][1], y[3][0], y[3][1]};
      } else {
        // (past the caches: 65.5 k rows of 8 x 128 81 us through them, 51 past them)
        __builtin_nontemporal_store(uint4v{pack2(y[0][0], y[0][1]), pack2(y[1][0], y[1][1]), pack2(y[2][0], y[2][1]), pack2(y[3][0], y[3][1])},
                                    (uint4v*)((bf16_t*)p.side[s].rows + at));
      }
    }
}

bool head_dim_taken(int d) {
  switch (d) {
    case 8: case 16: case 24: case 32: case 48: case 64: case 96: case 128: case 192: case 256: return true;
    default: return false;
  }
}

}  // namespace

int serve_check_pages(const HstuKvPages& g) {
  if (!g.k_codes || !g.k_scales || !g.v_codes || !g.v_scales) return serve_fail(HSTU_SERVE_ERR_NULL, "codes or scales are null");
  if (g.B < 0 || g.H < 1 || g.n_pages < 0 || g.table_pages < 0) return serve_fail(HSTU_SERVE_ERR_SHAPE, "B=%d H=%d n_pages=%d table_pages=%d", g.B, g.H, g.n_pages, g.table_pages);
  if (g.B > 0 && g.table_pages > 0 && !g.page_table) return serve_fail(HSTU_SERVE_ERR_NULL, "page_table is null");
  if (g.bits != 4 && g.bits != 8) return serve_fail(HSTU_SERVE_ERR_SHAPE, "bits=%d: 4 or 8", g.bits);
  if (!head_dim_taken(g.d)) return serve_fail(HSTU_SERVE_ERR_SHAPE, "d=%d: 8, 16, 24, 32, 48, 64, 96, 128, 192 or 256", g.d);
  // (a head's part of a page stays within 32 bits)
  if (g.page_size < 32 || g.page_size % 32 || g.page_size > 1 << 20) return serve_fail(HSTU_SERVE_ERR_SHAPE, "page_size=%d: a multiple of 32, at most 2^20", g.page_size);
  for (const void* t : {g.k_codes, g.k_scales, g.v_codes, g.v_scales})
    if (!serve_aligned16(t)) return serve_fail(HSTU_SERVE_ERR_SHAPE, "codes and scales start on 16-byte boundaries");
  return HSTU_SERVE_OK;
}

namespace {

int kv_rows(const HstuKvRowsArgs* a, void* stream, bool write) {
  serve_clear_error();
  if (!a) return serve_fail(HSTU_SERVE_ERR_NULL, "args is null");
  if (a->struct_size != sizeof(HstuKvRowsArgs) || a->version != HSTU_SERVE_ABI_VERSION)
    return serve_fail(HSTU_SERVE_ERR_VERSION, "struct_size %u version %u, expected %zu and %d", a->struct_size, a->version, sizeof(HstuKvRowsArgs), HSTU_SERVE_ABI_VERSION);
  if (const int rc = serve_check_pages(a->pages)) return rc;
  if (a->dtype != HSTU_SERVE_BF16 && a->dtype != HSTU_SERVE_FP32) return serve_fail(HSTU_SERVE_ERR_SHAPE, "dtype %d", a->dtype);
  if (a->rows_per_seq < 0 || a->total_rows < 0) return serve_fail(HSTU_SERVE_ERR_SHAPE, "rows_per_seq=%d total_rows=%lld", a->rows_per_seq, (long long)a->total_rows);
  const HstuKvPages& g = a->pages;
  if (g.B == 0 || a->rows_per_seq == 0 || (a->offsets && a->total_rows == 0)) return HSTU_SERVE_OK;
  if (!a->starts || !a->k || !a->v) return serve_fail(HSTU_SERVE_ERR_NULL, "starts, k or v is null");
  const int64_t unit = a->dtype == HSTU_SERVE_FP32 ? 4 : 8;       // elements of 16 bytes
  for (const void* t : {a->k, a->v})
    if (!serve_aligned16(t)) return serve_fail(HSTU_SERVE_ERR_SHAPE, "k and v start on 16-byte boundaries");
  for (const int64_t s : {a->k_stride_t, a->k_stride_h, a->v_stride_t, a->v_stride_h, a->offsets ? (int64_t)0 : a->k_stride_b, a->offsets ? (int64_t)0 : a->v_stride_b})
    if (s % unit) return serve_fail(HSTU_SERVE_ERR_SHAPE, "a stride of %lld elements: rows start on 16-byte boundaries", (long long)s);
  const int64_t tiles = ((int64_t)a->rows_per_seq + 31 + 31) / 32;   // (the first place may lie anywhere in its 32)
  if (tiles * g.H > SERVE_THREADS / 256 / g.B) return serve_fail(HSTU_SERVE_ERR_SHAPE, "%lld x %d x %d tiles are too many for one call", (long long)tiles, g.H, g.B);
  Params p;
  p.g = g;
  p.side[0] = Side{(uint8_t*)g.k_codes, (uint8_t*)g.k_scales, a->k, a->k_stride_b, a->k_stride_t, a->k_stride_h};
  p.side[1] = Side{(uint8_t*)g.v_codes, (uint8_t*)g.v_scales, a->v, a->v_stride_b, a->v_stride_t, a->v_stride_h};
  p.starts = a->starts;
  p.offsets = a->offsets;
  p.total = a->total_rows;
  p.per_seq = a->rows_per_seq;
  p.tiles = (int32_t)tiles;
  const uint32_t grid = (uint32_t)(tiles * g.H * g.B);
  hipStream_t st = (hipStream_t)stream;
#define KV_LAUNCH(BITS, F32, LPR)                                                        \
  do {                                                                                   \
    if (write) hstu_kv_write_kernel<BITS, F32, LPR><<<grid, threads_of(LPR), 0, st>>>(p);        \
    else hstu_kv_read_kernel<BITS, F32, LPR><<<grid, threads_of(LPR), 0, st>>>(p);               \
  } while (0)
#define KV_WIDTH(BITS, F32)                              \
  do {                                                   \
    if (g.d <= 32) KV_LAUNCH(BITS, F32, 4);              \
    else if (g.d <= 64) KV_LAUNCH(BITS, F32, 8);         \
    else if (g.d <= 128) KV_LAUNCH(BITS, F32, 16);       \
    else KV_LAUNCH(BITS, F32, 32);                       \
  } while (0)
  const bool f32 = a->dtype == HSTU_SERVE_FP32;
  if (g.bits == 4) { if (f32) KV_WIDTH(4, true); else KV_WIDTH(4, false); }
  else { if (f32) KV_WIDTH(8, true); else KV_WIDTH(8, false); }
#undef KV_WIDTH
#undef KV_LAUNCH
  return serve_launched(write ? "hstu_kv_write" : "hstu_kv_read");
}

}  // namespace

extern "C" {

int hstu_kv_write(const HstuKvRowsArgs* args, void* stream) { return kv_rows(args, stream, true); }
int hstu_kv_read(const HstuKvRowsArgs* args, void* stream) { return kv_rows(args, stream, false); }
int hstu_serve_abi_version(void) { return HSTU_SERVE_ABI_VERSION; }
const char* hstu_serve_last_error(void) { return g_err; }

}
