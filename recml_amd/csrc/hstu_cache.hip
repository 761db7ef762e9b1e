// The pages of a cache of keys and values in 4 or 8 bits, for gfx950 (MI355X): see include/hstu_serve.h.
//
//   hstu_kv_write   rows of new events -> codes and block exponents
//   hstu_kv_read    codes and exponents -> rows
//
// Both are passes over memory.  One workgroup takes 32 places of one (sequence, head): page sizes are multiples of 32 and
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
constexpr int THREADS = 256;

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

template <bool F32>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&x)[8]) {
  if constexpr (F32) {
    const floatx4* s = (const floatx4*)((const float*)base + at);
    const floatx4 a = s[0], b = s[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
  } else {
    unpack8(*(const uint4*)((const bf16_t*)base + at), x);
  }
}

// LPR lanes per row (8 values each); rows r, r + THREADS / LPR, ... of the tile.
template <int BITS, bool F32, int LPR>
__global__ __launch_bounds__(THREADS) void hstu_kv_write_kernel(const Params p) {
  constexpr int ROWS = THREADS / LPR;
  const int d = p.g.d, H = p.g.H, page = p.g.page_size;
  const int h = blockIdx.x % H, tile = blockIdx.x / H % p.tiles, b = blockIdx.x / H / p.tiles;
  const Side s = p.side[blockIdx.y];
  int64_t first;
  int count;
  rows_of(p, b, &first, &count);
  const int64_t start = p.starts[b];
  // places of the tile: whole multiples of 32, the first one at or below `start` (which may be negative)
  const int64_t base = (start - (((start % TILE) + TILE) % TILE)) + (int64_t)tile * TILE;
  if (base >= start + count) return;
  const int64_t row0 = kv_row(p.g, b, base);
  if (row0 < 0) return;
  const int lane = threadIdx.x % LPR;
  const int blocks = (d + 31) / 32, row_bytes = d * BITS / 8;
  const int64_t head0 = row0 + (int64_t)h * page;               // row of the tile's first place in its head's rows
  // (codes: rows of row_bytes; exponents: [page, head, block, slot])
  const int64_t page_head = (row0 / page) + h, slot0 = row0 % page;
  for (int r = threadIdx.x / LPR; r < TILE; r += ROWS) {
    const int64_t t = base + r - start;
    const bool there = t >= 0 && t < count && lane * 8 < d;
    float x[8] = {};
    if (there) load8<F32>(s.rows, (p.offsets ? 0 : (int64_t)b * s.sb) + (first + t) * s.st + (int64_t)h * s.sh + lane * 8, x);
    float top = 0.f;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t m = __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu;
      bad |= m >= 0x7f800000u;
      top = fmaxf(top, __builtin_bit_cast(float, m));
    }
    // a block's four lanes, then the row's
#pragma unroll
    for (int m = 1; m < 4 && m < LPR; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
#pragma unroll
    for (int m = 1; m < LPR; m <<= 1) bad |= __shfl_xor(bad, m, 64);
    // the exponent: floor(log2 top) less the largest code's, one more where top is past the middle above that code
    const uint32_t bits = __builtin_bit_cast(uint32_t, top);
    constexpr int TOP_EXP = BITS == 4 ? 2 : 8;
    constexpr uint32_t PAST = BITS == 4 ? 0x600000u : 0x680000u;      // mantissas of 1.75 and 1.8125
    int e = (int)(bits >> 23) - TOP_EXP + ((bits & 0x7fffffu) > PAST ? 1 : 0);
    constexpr int MOST = BITS == 4 ? 252 : 246;                        // (no code stands for more than fp32 holds: such rows saturate)
    e = e < 1 ? 1 : e > MOST ? MOST : e;                               // (top = 0 too)
    const float inverse = power_of((uint32_t)(254 - e));
    uint32_t code[2] = {0, 0};
    if (!bad) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = x[i] * inverse, m = __builtin_fabsf(y);
        if constexpr (BITS == 4) {
          // the grid's steps are 1/2 below 2, 1 below 4 and 2 from there: rint at each is to the nearest code, ties to even
          const float c = m < 2.f ? __builtin_rintf(2.f * m) : m < 4.f ? __builtin_rintf(m) + 2.f : fminf(__builtin_rintf(0.5f * m) + 4.f, 7.f);
          code[0] |= ((uint32_t)c | ((__builtin_bit_cast(uint32_t, y) >> 28) & 8u)) << (4 * i);
        } else {
          const float z = fminf(fmaxf(y, -448.f), 448.f);
          const int byte = __builtin_amdgcn_cvt_pk_fp8_f32(z, z, 0, false) & 0xff;
          code[i / 4] |= (uint32_t)byte << (8 * (i % 4));
        }
      }
    }
    if (!there) continue;
    uint8_t* to = s.codes + (head0 + r) * row_bytes + lane * BITS;
    if constexpr (BITS == 4) *(uint32_t*)to = code[0];
    else *(uint2*)to = uint2{code[0], code[1]};
    if (lane % 4 == 0) s.scales[(page_head * blocks + lane / 4) * page + slot0 + r] = (uint8_t)(bad ? 255 : e);
  }
}

template <int BITS, bool F32, int LPR>
__global__ __launch_bounds__(THREADS) void hstu_kv_read_kernel(const Params p) {
  constexpr int ROWS = THREADS / LPR;
  const int d = p.g.d, H = p.g.H, page = p.g.page_size;
  const int h = blockIdx.x % H, tile = blockIdx.x / H % p.tiles, b = blockIdx.x / H / p.tiles;
  const Side s = p.side[blockIdx.y];
  int64_t first;
  int count;
  rows_of(p, b, &first, &count);
  const int64_t start = p.starts[b];
  const int64_t base = (start - (((start % TILE) + TILE) % TILE)) + (int64_t)tile * TILE;
  if (base >= start + count) return;
  const int64_t row0 = kv_row(p.g, b, base);
  const int lane = threadIdx.x % LPR;
  if (lane * 8 >= d) return;
  const int blocks = (d + 31) / 32, row_bytes = d * BITS / 8;
  const int64_t head0 = row0 + (int64_t)h * page, page_head = (row0 / page) + h, slot0 = row0 % page;
  for (int r = threadIdx.x / LPR; r < TILE; r += ROWS) {
    const int64_t t = base + r - start;
    if (t < 0 || t >= count) continue;
    float y[8] = {};
    if (row0 >= 0) {
      const uint8_t* from = s.codes + (head0 + r) * row_bytes + lane * BITS;
      const uint32_t e = s.scales[(page_head * blocks + lane / 4) * page + slot0 + r];
      const float power = e == 255u ? __builtin_nanf("") : power_of(e);
      if constexpr (BITS == 4) {
        const uint32_t w = *(const uint32_t*)from;
        const floatx2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1),
                      c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
        y[0] = a[0]; y[1] = a[1]; y[2] = b2[0]; y[3] = b2[1]; y[4] = c[0]; y[5] = c[1]; y[6] = f[0]; y[7] = f[1];
      } else {
        const uint2 w = *(const uint2*)from;
        const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false), b2 = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true),
                      c = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false), f = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
        y[0] = a[0]; y[1] = a[1]; y[2] = b2[0]; y[3] = b2[1]; y[4] = c[0]; y[5] = c[1]; y[6] = f[0]; y[7] = f[1];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= power;
    }
    const int64_t at = (p.offsets ? 0 : (int64_t)b * s.sb) + (first + t) * s.st + (int64_t)h * s.sh + lane * 8;
    if constexpr (F32) {
      floatx4* to = (floatx4*)((float*)s.rows + at);
      to[0] = floatx4{y[0], y[1], y[2], y[3]};
      to[1] = floatx4{y[4], y[5], y[6], y[7]};
    } else {
      *(uint4*)((bf16_t*)s.rows + at) = uint4{pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7])};
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
  if (g.page_size < 32 || g.page_size % 32) return serve_fail(HSTU_SERVE_ERR_SHAPE, "page_size=%d: a multiple of 32", g.page_size);
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
  if (tiles * g.H > 0x7fffffffll || tiles * g.H * g.B > 0x7fffffffll) return serve_fail(HSTU_SERVE_ERR_SHAPE, "%lld x %d x %d tiles are too many for one call", (long long)tiles, g.H, g.B);
  Params p;
  p.g = g;
  p.side[0] = Side{(uint8_t*)g.k_codes, (uint8_t*)g.k_scales, a->k, a->k_stride_b, a->k_stride_t, a->k_stride_h};
  p.side[1] = Side{(uint8_t*)g.v_codes, (uint8_t*)g.v_scales, a->v, a->v_stride_b, a->v_stride_t, a->v_stride_h};
  p.starts = a->starts;
  p.offsets = a->offsets;
  p.total = a->total_rows;
  p.per_seq = a->rows_per_seq;
  p.tiles = (int32_t)tiles;
  const dim3 grid((uint32_t)(tiles * g.H * g.B), 2);
  hipStream_t st = (hipStream_t)stream;
#define KV_LAUNCH(BITS, F32, LPR)                                                        \
  do {                                                                                   \
    if (write) hstu_kv_write_kernel<BITS, F32, LPR><<<grid, THREADS, 0, st>>>(p);        \
    else hstu_kv_read_kernel<BITS, F32, LPR><<<grid, THREADS, 0, st>>>(p);               \
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
