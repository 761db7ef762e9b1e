// The product of rows in 8 bits with a weight in 8 bits on the scaled matrix instructions of gfx950: see include/hstu_rows8.h.
//
//   out[m, n] = act(sum_b 2^(ex[m, b] - 127) 2^(ew[n, b] - 127) sum_{k in block b} x[m, k] w[n, k] + c[m, n] + bias[n])
//
// A block's powers are the scale operands of v_mfma_scale_f32_32x32x64_f8f6f4, so the sum over the blocks stays in its accumulators: no
// step between blocks.  Both operands lie along the contraction.
//
// What those instructions round: of each eight neighbouring products they cut every one, toward zero, to a grid of 2^-13 of the largest of
// the eight (beside 2^16 a product of 28 counts as 24, one of 7 as none), then add in fp32, the accumulator included.  That is four bits more
// than a bf16 result keeps, and 2e-5 of a result in the mean square beside 1.7e-3 of its rounding, so bf16 results are made this way (1.5 % of them
// are then the exact value's other neighbour).  An fp32 result is not: its codes
// become bf16 values, exactly (under the smallest two exponents to the nearest multiple of bf16's least value, 2^-133), by a conversion that takes
// the powers along, and go through bf16's instruction, whose sums are fp32's (results
// are off by 1e-8 of themselves at 200 values a row to 1e-7 at 4096), at half the rate.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#include "hstu_rows8_common.h"

namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

struct GemmParams {
  const uint8_t *x, *w;              // codes
  const uint8_t *xe, *we;            // exponents
  void* out;
  const void* c;
  const void* bias;
  int64_t out_stride, c_stride;
  int32_t rows, cols;                // of the output: rows of x, rows of w
  int32_t blocks;                    // of 128 along the contraction
  int32_t row_tiles, col_tiles;
  int32_t activation, vec;           // vec: out and c are whole vectors of 16 bytes everywhere
};

#define ROWS8_WAIT_VMCNT(n) __builtin_amdgcn_s_waitcnt((((n) & 15) | ((((n) >> 4) & 3) << 14)) | 0x0F70)

// Loads straight into LDS: 16 or 4 bytes a lane, side by side from the given place on.
__device__ __forceinline__ void lds_dma16(const uint8_t* base, uint32_t off, uint32_t lds) {
  const uint32_t to = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void lds_dma4(const uint8_t* base, uint32_t off, uint32_t lds) {
  const uint32_t to = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(to), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ const uint8_t* scalar_ptr(const uint8_t* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const uint8_t*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

// x sigmoid(x) by the hardware's exp2 and reciprocal (1 ulp each)
__device__ __forceinline__ float silu(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

template <bool F32>
__device__ __forceinline__ float value_of(const void* base, int64_t at) {
  return F32 ? ((const float*)base)[at] : (float)((const bf16_t*)base)[at];
}

// Eight values of the output's type side by side, at any place that the type may have: the wide accesses of this chip need no more.
typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t words2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float floats4 __attribute__((ext_vector_type(4), aligned(4)));
template <bool F32>
__device__ __forceinline__ void row_load8(const void* base, int64_t at, float (&f)[8]) {
  if constexpr (F32) {
    const floats4* const from = (const floats4*)((const float*)base + at);
    const floatx4 lo = (floatx4)from[0], hi = (floatx4)from[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = lo[i]; f[4 + i] = hi[i]; }
  } else {
    unpack8((uint4v)*(const words4*)((const bf16_t*)base + at), f);
  }
}
template <bool F32>
__device__ __forceinline__ void row_store8(void* base, int64_t at, const float (&f)[8]) {
  if constexpr (F32) {
    floats4* const to = (floats4*)((float*)base + at);
    to[0] = floats4{f[0], f[1], f[2], f[3]};
    to[1] = floats4{f[4], f[5], f[6], f[7]};
  } else {
    *(words4*)((bf16_t*)base + at) = pack8(f);      // (past the L2s, as the bf16 products store large outputs, it is no faster)
  }
}

// Four values of a row added, from column `at` on; none past `cols`.
template <bool F32>
__device__ __forceinline__ void add4(const void* base, int64_t row, int at, int cols, floatx4& y) {
  if (at + 4 <= cols) {
    if constexpr (F32) {
      const floatx4 v = (floatx4)*(const floats4*)((const float*)base + row + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += v[i];
    } else {
      const words2 v = *(const words2*)((const bf16_t*)base + row + at);
      y[0] += __builtin_bit_cast(float, v.x << 16);
      y[1] += __builtin_bit_cast(float, v.x & 0xffff0000u);
      y[2] += __builtin_bit_cast(float, v.y << 16);
      y[3] += __builtin_bit_cast(float, v.y & 0xffff0000u);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i < cols) y[i] += value_of<F32>(base, row + at + i);
}

// Eight of a lane's 32 codes as the values that they stand for in bf16: exact from an exponent of 3 on.
__device__ __forceinline__ bf16x8 values8(const intx8& codes, int q, float power) {
  const uint32_t lo = (uint32_t)codes[2 * q], hi = (uint32_t)codes[2 * q + 1];
  struct { bf16x2 v[4]; } all = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, true),
                                 __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, true)};
  return __builtin_bit_cast(bf16x8, all);
}

// LDS of a stage of one set of waves, and of a workgroup (what the epilogue and the sum over the sets exchange takes the stages' place).
constexpr int stage_bytes(int tm, int tn) { return (tm + tn) * (BLOCK + 4); }
constexpr int lds_bytes(int mb, int nb, int wm, int wn, int stages, int ks) {
  const int ring = stages * ks * stage_bytes(32 * mb * wm, 32 * nb * wn), out = wm * wn * (32 * (32 * nb * 4 + 16) + (ks - 1) * nb * mb * 4096);
  return ring > out ? ring : out;
}

// Which tile a workgroup has; false: none.  Workgroups go to the eight XCDs in turn: each XCD takes a run of the tiles, which go by eight
// rows of tiles at a time.
__device__ __forceinline__ bool tile_of(const GemmParams& g, int* rt, int* ct) {
  const int all = g.row_tiles * g.col_tiles, each = (all + 7) >> 3;
  const int tile = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= each || tile >= all) return false;
  const int band = tile / (8 * g.col_tiles), in_band = tile - band * 8 * g.col_tiles;
  const int high = g.row_tiles - 8 * band < 8 ? g.row_tiles - 8 * band : 8;
  *ct = in_band / high;
  *rt = 8 * band + in_band - *ct * high;
  return true;
}

// A wave's sums on their way out: blocks of 32 rows x 32 NB columns from (m0, n0) on, through the wave's own LDS (fp32, rows 16 bytes apart
// from a multiple of 128), then pieces of 8 columns of a row per lane, wherever rows begin and end: 911 x 1218 to 11469 23 us, to 11472 23, by single
// values 32; 1237 x 1001 to 777 in fp32 with a residual 9.1, to 776 9.0, by single values 11.
template <int MB, int NB, bool F32>
__device__ __forceinline__ void tile_out(const GemmParams& g, const floatx16 (&acc)[NB][MB], uint8_t* stage, int m0, int n0) {
  const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
  constexpr int W = 32 * NB, PITCH = W * 4 + 16;
  auto put = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < NB; ++a)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *(floatx4*)(stage + l32 * PITCH + (32 * a + 8 * q4 + 4 * hh) * 4) =
            floatx4{acc[a][b][4 * q4], acc[a][b][4 * q4 + 1], acc[a][b][4 * q4 + 2], acc[a][b][4 * q4 + 3]};
    __builtin_amdgcn_wave_barrier();
  };
  if (n0 + 8 > g.cols) {                               // fewer columns than a piece: one a lane, 8 rows an instruction
    const int col = lane % 8, n = n0 + col;
    const bool in = n < g.cols;
    const float bias = g.bias && in ? value_of<F32>(g.bias, n) : 0.f;
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      put(b);
      const int mb = m0 + 32 * b + lane / 8;
      float cv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) cv[i] = g.c && in && mb + 8 * i < g.rows ? value_of<F32>(g.c, (int64_t)(mb + 8 * i) * g.c_stride + n) : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!in || mb + 8 * i >= g.rows) continue;
        float y = *(const float*)(stage + (8 * i + lane / 8) * PITCH + 4 * col) + cv[i] + bias;
        if (g.activation) y = silu(y);
        const int64_t to = (int64_t)(mb + 8 * i) * g.out_stride + n;
        if constexpr (F32) ((float*)g.out)[to] = y;
        else ((bf16_t*)g.out)[to] = (bf16_t)y;
      }
      __builtin_amdgcn_wave_barrier();
    }
    return;
  }
  constexpr int LPR = W / 8, RPI = 64 / LPR, PIECES = 32 / RPI;        // lanes per row, rows per instruction
  const int rr = lane / LPR, cc = lane - rr * LPR;
  // a row's last piece, if it is not whole, is its last eight columns (some written twice, with the same values)
  const bool part = n0 + W > g.cols && g.cols % 8;
  const bool has = n0 + 8 * cc < g.cols;
  const int n = n0 + 8 * cc < g.cols - 8 ? n0 + 8 * cc : has ? g.cols - 8 : n0 + 8 * cc, col = n - n0;
  float bias[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) bias[i] = 0.f;
  if (g.bias && has) row_load8<F32>(g.bias, n, bias);
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    put(b);
    float y[PIECES][8];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const uint8_t* at = stage + (RPI * i + rr) * PITCH + 4 * col;
      if (part) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = ((const float*)at)[e];
        continue;
      }
      const floatx4 lo = *(const floatx4*)at, hi = *(const floatx4*)(at + 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) { y[i][e] = lo[e]; y[i][4 + e] = hi[e]; }
    }
    const int mb = m0 + 32 * b + rr;      // the lane's row of piece 0
    auto inside = [&](int i) __attribute__((always_inline)) { return has && mb + RPI * i < g.rows; };
    if (g.c) {
      float cv[PIECES][8];
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) cv[i][e] = 0.f;
        if (inside(i)) row_load8<F32>(g.c, (int64_t)(mb + RPI * i) * g.c_stride + n, cv[i]);
      }
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] += cv[i][e];
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) y[i][e] += bias[e];
    if (g.activation) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = silu(y[i][e]);
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
      if (inside(i)) row_store8<F32>(g.out, (int64_t)(mb + RPI * i) * g.out_stride + n, y[i]);
    __builtin_amdgcn_wave_barrier();
  }
}

// One workgroup: a tile of 32 MB WM rows of x by 32 NB WN rows of w (output columns), WM x WN waves of 32 MB x 32 NB.  The contraction runs
// in stages of one block of 128 through an LDS ring filled by direct loads; a stage is the codes of both operands and their rows' exponents
// (the four of a group at once: one byte of them is read).  The product is formed transposed (columns as the matrix instruction's rows): a
// lane then holds four consecutive columns of one output row.
//   A row's 128 bytes lie in LDS as eight 16-byte chunks, chunk c of row r at c ^ (r / 2 % 8): 16 rows reach all 64 banks.  Which
// contraction elements a lane holds does not matter as long as both operands' lanes hold the same ones.
//   KS > 1: as many sets of waves, each with the blocks of its turn; their sums are added in LDS in the sets' order.
//   For results in bf16 the tiles are of 128 x 128 and less (hstu_rows8_turns_kernel has the larger ones).
template <int MB, int NB, int WM, int WN, int STAGES, int KS, bool F32>
__global__ __launch_bounds__(64 * WM * WN * KS) void hstu_rows8_gemm_kernel(const GemmParams g) {
  constexpr int TM = 32 * MB * WM, TN = 32 * NB * WN, WAVES = WM * WN;
  constexpr int OUT_BYTES = 32 * (32 * NB * 4 + 16);            // of a wave, in tile_out
  constexpr int X_BYTES = TM * BLOCK, CODES = (TM + TN) * BLOCK, PART = stage_bytes(TM, TN), STAGE = KS * PART;
  constexpr int LX = TM / 8 / WAVES, LW = TN / 8 / WAVES, LE = (TM + TN) / 64, LEW = (LE + WAVES - 1) / WAVES;      // direct loads of 8 rows; of 64 rows' exponents
  static_assert(LX * 8 * WAVES == TM && LW * 8 * WAVES == TN && TM % 64 == 0 && TN % 64 == 0, "whole loads a wave");
  constexpr int NLOAD = LX + LW + LEW;
  static_assert(STAGES >= 2 && (STAGES - 1) * NLOAD <= 63, "vmcnt range");
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const uint32_t smem_lds = __builtin_amdgcn_groupstaticsize();
  const int tid = threadIdx.x, lane = tid & 63;
  const int all_w = __builtin_amdgcn_readfirstlane(tid >> 6), ks = all_w / WAVES, w = all_w % WAVES;      // KS sets of waves, a block each
  const int l32 = lane & 31, hh = lane >> 5;

  int rt, ct;
  if (!tile_of(g, &rt, &ct)) return;
  const int m0 = rt * TM, n0 = ct * TN, nt = (g.blocks + KS - 1) / KS;

  // ---- what each lane loads: piece i of an operand is 8 rows, lane l of it the 16 bytes at row l / 8, place l % 8.  Rows past an operand's
  // end are its last one (what they give is not stored).
  const int64_t pitch = (int64_t)g.blocks * BLOCK;
  uint32_t xo[LX], wo[LW];
#pragma unroll
  for (int i = 0; i < LX; ++i) {
    const int r = 8 * (w * LX + i) + (lane >> 3), at = m0 + r < g.rows ? r : g.rows - 1 - m0;
    xo[i] = (uint32_t)(at * (int)pitch + 16 * ((lane & 7) ^ ((r >> 1) & 7)));
  }
#pragma unroll
  for (int i = 0; i < LW; ++i) {
    const int r = 8 * (w * LW + i) + (lane >> 3), at = n0 + r < g.cols ? r : g.cols - 1 - n0;
    wo[i] = (uint32_t)(at * (int)pitch + 16 * ((lane & 7) ^ ((r >> 1) & 7)));
  }
  // (more waves than pieces of exponents: some load the same)
  uint32_t eo[LEW], e_to[LEW];
  const uint8_t* e_base[LEW];
  int64_t e_step[LEW];
#pragma unroll
  for (int i = 0; i < LEW; ++i) {
    const int piece = (w + WAVES * i) % LE;
    const bool of_x = 64 * piece < TM;
    const int row = (of_x ? 64 * piece : 64 * piece - TM) + lane, last = of_x ? g.rows - 1 - m0 : g.cols - 1 - n0;
    eo[i] = 4u * (uint32_t)(row < last ? row : last);
    e_to[i] = CODES + 256u * piece;
    e_base[i] = scalar_ptr(of_x ? g.xe + (int64_t)m0 * 4 : g.we + (int64_t)n0 * 4);
    e_step[i] = 4 * (int64_t)(of_x ? g.rows : g.cols);
  }
  const uint8_t* x_base = scalar_ptr(g.x + (int64_t)m0 * pitch);
  const uint8_t* w_base = scalar_ptr(g.w + (int64_t)n0 * pitch);
  int block = ks;                                               // of the next stage to load (past the last one that is loaded again, and not used)
  auto issue = [&](int st) __attribute__((always_inline)) {
    const uint32_t base = smem_lds + (uint32_t)(st * STAGE + ks * PART);
    const int at = block < g.blocks ? block : g.blocks - 1;
    const uint8_t *const x_from = x_base + at * BLOCK, *const w_from = w_base + at * BLOCK;
#pragma unroll
    for (int i = 0; i < LX; ++i) lds_dma16(x_from, xo[i], base + 1024u * (w * LX + i));
#pragma unroll
    for (int i = 0; i < LW; ++i) lds_dma16(w_from, wo[i], base + X_BYTES + 1024u * (w * LW + i));
#pragma unroll
    for (int i = 0; i < LEW; ++i) lds_dma4(e_base[i] + (at >> 2) * e_step[i], eo[i], base + e_to[i]);
    block += KS;
  };

  // ---- fragments: lane (row l32 of a block of 32, half hh) holds two chunks of each half of the row's 128 bytes
  const int wm = w % WM, wn = w / WM;
  uint32_t fo[2][2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h) fo[s][h] = (uint32_t)(l32 * BLOCK + 16 * ((4 * s + 2 * hh + h) ^ ((l32 >> 1) & 7)));
  auto frag = [&](int st, int row0, int s) __attribute__((always_inline)) {
    const uint8_t* const at = smem + st * STAGE + ks * PART + row0 * BLOCK;
    struct { uint4v a, b; } both = {*(const uint4v*)(at + fo[s][0]), *(const uint4v*)(at + fo[s][1])};
    return __builtin_bit_cast(intx8, both);
  };
  auto w_frag = [&](int st, int a, int s) __attribute__((always_inline)) { return frag(st, TM + 32 * (wn * NB + a), s); };
  auto x_frag = [&](int st, int b, int s) __attribute__((always_inline)) { return frag(st, 32 * (wm * MB + b), s); };
  int xs[MB], ws[NB];
  auto scales = [&](int st, int t) __attribute__((always_inline)) {
    const uint8_t* const at = smem + st * STAGE + ks * PART + CODES + 4 * l32 + ((t * KS + ks) & 3);
#pragma unroll
    for (int a = 0; a < NB; ++a) ws[a] = at[4 * (TM + 32 * (wn * NB + a))];
#pragma unroll
    for (int b = 0; b < MB; ++b) xs[b] = at[4 * 32 * (wm * MB + b)];
  };

  floatx16 acc[NB][MB];
#pragma unroll
  for (int a = 0; a < NB; ++a)
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;

#pragma unroll
  for (int t = 0; t < STAGES; ++t)
    if (t < nt) issue(t);
  // (stages younger than the one waited for: as many as the ring has, or fewer near the end, where the wait is for all)
  if (nt >= STAGES) ROWS8_WAIT_VMCNT((STAGES - 1) * NLOAD);
  else ROWS8_WAIT_VMCNT(0);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  int st = 0;
  for (int t = 0; t < nt; ++t) {
    if (KS == 1 || t * KS + ks < g.blocks) {
    scales(st, t);
    float wp[NB], xp[MB];
    if constexpr (F32) {
#pragma unroll
      for (int a = 0; a < NB; ++a) wp[a] = power_of((uint32_t)ws[a]);
#pragma unroll
      for (int b = 0; b < MB; ++b) xp[b] = power_of((uint32_t)xs[b]);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      intx8 wf[NB], xf[MB];
#pragma unroll
      for (int a = 0; a < NB; ++a) wf[a] = w_frag(st, a, s);
#pragma unroll
      for (int b = 0; b < MB; ++b) xf[b] = x_frag(st, b, s);
      if constexpr (F32) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          bf16x8 wv[NB], xv[MB];
#pragma unroll
          for (int a = 0; a < NB; ++a) wv[a] = values8(wf[a], q, wp[a]);
#pragma unroll
          for (int b = 0; b < MB; ++b) xv[b] = values8(xf[b], q, xp[b]);
#pragma unroll
          for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int a = 0; a < NB; ++a) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wv[a], xv[b], acc[a][b], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int a = 0; a < NB; ++a) acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[a], xf[b], acc[a][b], 0, 0, 0, ws[a], 0, xs[b]);
      }
    }
    }
    // everyone's last read of this stage is done, and the next stage's loads are here
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + STAGES <= nt) ROWS8_WAIT_VMCNT((STAGES - 2) * NLOAD);
    else ROWS8_WAIT_VMCNT(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (t + STAGES < nt) issue(st);
    st = st + 1 >= STAGES ? 0 : st + 1;
  }

  if constexpr (KS > 1) {
    // the sets' sums, added in their order
    floatx4* const sums = (floatx4*)(smem + WAVES * OUT_BYTES);
    if (ks > 0) {
#pragma unroll
      for (int a = 0; a < NB; ++a)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            sums[((((ks - 1) * WAVES + w) * NB + a) * MB + b) * 256 + 64 * q + lane] =
                floatx4{acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]};
    }
    __syncthreads();
    if (ks > 0) return;
#pragma unroll
    for (int i = 0; i < KS - 1; ++i)
#pragma unroll
      for (int a = 0; a < NB; ++a)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const floatx4 v = sums[(((i * WAVES + w) * NB + a) * MB + b) * 256 + 64 * q + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[a][b][4 * q + e] += v[e];
          }
  }
  tile_out<MB, NB, F32>(g, acc, smem + w * OUT_BYTES, m0 + 32 * MB * wm, n0 + 32 * NB * wn);
}

// The same product where there is work for tiles of 256 x 256 and a contraction to stream.  Eight waves of 128 x 64 in two halves, one wave of
// each to a SIMD, that take turns: while one half forms a stage's products the other reads its fragments of the next from LDS and asks for
// more of it, and a barrier changes them over.  So the matrix pipe and LDS are both at work all the time, where waves that go in step leave
// each idle in turn.  16384 x 8192 by 8192 in 833 us (2640 TFLOP/s; in step 878), 8192 of each 414 (in step 425), 16384 x 2048 to 8192 246
// (258).  What bounds it is power: the matrix pipe is at work two thirds of the time, at a clock of 1.8 GHz that waves in step, 58 %, find at
// 2.0.  Four waves of 128 x 128, which read a third less of LDS, one to a SIMD, took 958 as the compiler schedules them.
__global__ __launch_bounds__(512, 2) void hstu_rows8_turns_kernel(const GemmParams g) {
  constexpr int T = 256, X_BYTES = T * BLOCK, CODES = 2 * X_BYTES, STAGE = stage_bytes(T, T);
  constexpr int L = T / 8 / 8, NLOAD = 2 * L + 1;              // direct loads of 8 rows a wave and operand; of 64 rows' exponents
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const uint32_t smem_lds = __builtin_amdgcn_groupstaticsize();
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  int rt, ct;
  if (!tile_of(g, &rt, &ct)) return;
  const int m0 = rt * T, n0 = ct * T, nt = g.blocks;

  // ---- what each lane loads, as hstu_rows8_gemm_kernel has it
  const int64_t pitch = (int64_t)g.blocks * BLOCK;
  uint32_t xo[L], wo[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int r = 8 * (w * L + i) + (lane >> 3);
    const uint32_t chunk = 16 * ((lane & 7) ^ ((r >> 1) & 7));
    xo[i] = (uint32_t)((m0 + r < g.rows ? r : g.rows - 1 - m0) * (int)pitch) + chunk;
    wo[i] = (uint32_t)((n0 + r < g.cols ? r : g.cols - 1 - n0) * (int)pitch) + chunk;
  }
  const bool of_x = w < 4;
  const int e_row = 64 * (w & 3) + lane, e_last = of_x ? g.rows - 1 - m0 : g.cols - 1 - n0;
  const uint32_t eo = 4u * (uint32_t)(e_row < e_last ? e_row : e_last);
  const uint8_t* x_base = scalar_ptr(g.x + (int64_t)m0 * pitch);
  const uint8_t* w_base = scalar_ptr(g.w + (int64_t)n0 * pitch);
  const uint8_t* e_base = scalar_ptr(of_x ? g.xe + (int64_t)m0 * 4 : g.we + (int64_t)n0 * 4);
  const int64_t e_step = 4 * (int64_t)(of_x ? g.rows : g.cols);
  int loaded = 0;                                               // stages asked for
  auto issue_one = [&](int st, int i) __attribute__((always_inline)) {
    const uint32_t base = smem_lds + (uint32_t)st * STAGE;
    if (i < L) lds_dma16(x_base, xo[i < L ? i : 0], base + 1024u * (w * L + i));
    else if (i < 2 * L) lds_dma16(w_base, wo[i < L ? 0 : i < 2 * L ? i - L : 0], base + X_BYTES + 1024u * (w * L + i - L));
    else {
      lds_dma4(e_base, eo, base + CODES + 256u * w);
      // (past the last block it is loaded again, into a place that nobody reads)
      const bool more = ++loaded < nt;
      x_base += more ? BLOCK : 0;
      w_base += more ? BLOCK : 0;
      e_base += more && (loaded & 3) == 0 ? e_step : 0;
    }
  };
  auto issue = [&](int st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NLOAD; ++i) issue_one(st, i);
  };

  const int wm = w & 1, wn = w >> 1;
  uint32_t fo[2][2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h) fo[s][h] = (uint32_t)(l32 * BLOCK + 16 * ((4 * s + 2 * hh + h) ^ ((l32 >> 1) & 7)));
  intx8 wf[2][2], xf[2][4];
  int ws[2], xs[4];
  auto take = [&](int st, int t) __attribute__((always_inline)) {
    const uint8_t* const at = smem + st * STAGE;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      auto frag = [&](int row0) __attribute__((always_inline)) {
        struct { uint4v a, b; } both = {*(const uint4v*)(at + row0 * BLOCK + fo[s][0]), *(const uint4v*)(at + row0 * BLOCK + fo[s][1])};
        return __builtin_bit_cast(intx8, both);
      };
#pragma unroll
      for (int a = 0; a < 2; ++a) wf[s][a] = frag(T + 64 * wn + 32 * a);
#pragma unroll
      for (int b = 0; b < 4; ++b) xf[s][b] = frag(128 * wm + 32 * b);
    }
    const uint8_t* const e = at + CODES + 4 * l32 + (t & 3);
#pragma unroll
    for (int a = 0; a < 2; ++a) ws[a] = e[4 * (T + 64 * wn + 32 * a)];
#pragma unroll
    for (int b = 0; b < 4; ++b) xs[b] = e[4 * (128 * wm + 32 * b)];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };

  floatx16 acc[2][4];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
  auto products = [&](auto refill_, int st) __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int s = i >> 3, b = (i >> 1) & 3, a = i & 1;
      acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[s][a], xf[s][b], acc[a][b], 0, 0, 0, ws[a], 0, xs[b]);
      asm volatile("" : "+v"(acc[a][b]));              // (the product stays here: the compiler would move it to where its result is used)
      if constexpr (decltype(refill_)::value) {
        __builtin_amdgcn_sched_barrier(0);
        if (i >= 2 && i < 2 + NLOAD) issue_one(st, i - 2);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto change = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // The first half reads stage t in turn 2 t and forms its products in turn 2 t + 1, the second half a turn later.  A stage's place is free
  // behind turn 2 t + 1: the first half asks for its share of stage t + 2 in turn 2 t + 2, beside the fragments of stage t + 1, the second half
  // in the same turn between the products of stage t.  Each waits for its share before the barrier behind turn 2 t + 3.
  issue(0);
  if (w >= 4) issue(1);
  if (w >= 4) ROWS8_WAIT_VMCNT(NLOAD);
  else ROWS8_WAIT_VMCNT(0);
  change();
  if (w < 4) {
    for (int t = 0; t < nt; ++t) {
      issue((t + 1) & 1);
      take(t & 1, t);
      change();
      products(std::false_type{}, 0);
      ROWS8_WAIT_VMCNT(0);
      change();
    }
    change();
  } else {
    change();
    for (int t = 0; t < nt; ++t) {
      take(t & 1, t);
      ROWS8_WAIT_VMCNT(0);
      change();
      products(std::true_type{}, t & 1);
      change();
    }
  }
  ROWS8_WAIT_VMCNT(0);
  __syncthreads();
  tile_out<4, 2, false>(g, acc, smem + w * (32 * (32 * 2 * 4 + 16)), m0 + 128 * wm, n0 + 64 * wn);
}

// f(0), f(1), ..., f(N - 1), each index a constant
template <int... I, typename F>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F&& f) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) { each_of(std::make_integer_sequence<int, N>{}, f); }

// The products of contractions of KB blocks with many outputs.  A wave keeps 32 rows of x as fragments in its registers, and the weight
// goes by in LDS, 32 of its columns and the whole contraction a stage.  A workgroup is eight waves; it takes a run of pieces of (256 rows,
// 64 columns), rows by rows: its ring of stages never empties, and x is read once, or twice where a tile is two workgroups'.
//   What bounds hstu_rows8_gemm_kernel at a short contraction is that a tile's loads, products, epilogue and stores take turns.  Here the
// products of a column block stand beside the epilogue of the one before it and a second wave of the SIMD beside both, and the stores go
// on meanwhile.  73728 x 512 to 2048 with SiLU 148 us in tiles of 256 x 256, 90 so (1710 TFLOP/s, 3.8 TB/s), plain 129 and 80; 16398 x 1024 to
// 4096 109 and 78; added to other rows, 73728 x 512 to 512 48 and 40; 73728 x 256 to 1024 56 and 41, x 64 to 256 16 and 13.  SiLU's two
// quarter-rate instructions a value are as much work as the products are.  Two blocks of 32 rows a wave halve the reads of LDS and are no
// faster (97 and 77).
enum { ROWS_PLAIN = 0, ROWS_SILU = 1, ROWS_ADD = 2 };            // (bits)
template <int KB, int OUT>
__global__ __launch_bounds__(512, 2) void hstu_rows8_rows_kernel(const GemmParams g) {
  constexpr int NS = 2 * KB, AHEAD = 1, STAGES = 3, GROUPS = (KB + 3) / 4, PITCH = KB * BLOCK;
  constexpr int CODES = 32 * PITCH, STAGE = CODES + 256;
  constexpr int LP = (4 * KB + 7) / 8, NLOAD = LP + 1;              // direct loads of 1 KB per wave and stage, and of exponents
  constexpr int STORES = 4;
  constexpr bool ADD = OUT & ROWS_ADD;
  static_assert(KB <= 8 && NS % (AHEAD + 1) == 0 && STAGES == 3, "fragments keep their registers from step to step");
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const uint32_t smem_lds = __builtin_amdgcn_groupstaticsize();
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;

  // this workgroup's run of pairs of column blocks, XCD by XCD
  const int pairs = g.cols >> 6;
  const int64_t all = (int64_t)g.row_tiles * pairs;
  const int64_t me = (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const int64_t first = all * me / gridDim.x, last = all * (me + 1) / gridDim.x;
  if (first >= last) return;
  // (scalars, which a division leaves in vector registers)
  int rt = __builtin_amdgcn_readfirstlane((int)(first / pairs)), pc = __builtin_amdgcn_readfirstlane((int)(first - (int64_t)rt * pairs));
  int todo = __builtin_amdgcn_readfirstlane((int)(last - first));

  // ---- the weight's stages: KB panels of 32 rows of 128 bytes, chunk c of row r at c ^ (r / 2 % 8); then the rows' exponents by groups
  uint32_t po[LP], p_to[LP];
#pragma unroll
  for (int i = 0; i < LP; ++i) {
    const int piece = (w + 8 * i) % (4 * KB), r = 8 * (piece & 3) + (lane >> 3);      // (more waves than pieces: some load the same)
    po[i] = (uint32_t)(r * PITCH + BLOCK * (piece >> 2) + 16 * ((lane & 7) ^ ((r >> 1) & 7)));
    p_to[i] = 1024u * piece;
  }
  const uint32_t eo = 4u * (uint32_t)l32 + (GROUPS > 1 ? (uint32_t)hh * 4u * (uint32_t)g.cols : 0u);
  int column = 64 * pc, left = 2 * todo;               // of the next stage to load; stages left to load
  auto load_stage = [&](int st) __attribute__((always_inline)) {
    const uint32_t base = smem_lds + (uint32_t)st * STAGE;
    const uint8_t* const from = scalar_ptr(g.w + (int64_t)column * PITCH);
#pragma unroll
    for (int i = 0; i < LP; ++i) lds_dma16(from, po[i], base + p_to[i]);
    lds_dma4(scalar_ptr(g.we + (int64_t)column * 4), eo, base + CODES);
    column = column + 32 == g.cols ? 0 : column + 32;
    --left;
  };
  uint32_t fo[2][2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h) fo[s][h] = (uint32_t)(l32 * BLOCK + 16 * ((4 * s + 2 * hh + h) ^ ((l32 >> 1) & 7)));
  intx8 f[AHEAD + 1];
  int we[2][GROUPS];                                   // of the stage at work, and of the one after it
  auto ask = [&](int st, auto s_) __attribute__((always_inline)) {
    constexpr int s = decltype(s_)::value;
    const uint8_t* const at = smem + st * STAGE + 4096 * (s / 2);
    struct { uint4v a, b; } both = {*(const uint4v*)(at + fo[s & 1][0]), *(const uint4v*)(at + fo[s & 1][1])};
    f[s % (AHEAD + 1)] = __builtin_bit_cast(intx8, both);
  };
  auto exponents = [&](int st, int to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) we[to][i] = *(const int*)(smem + st * STAGE + CODES + 128 * i + 4 * l32);
  };

  intx8 xf[NS];
  int xe[GROUPS];
  auto load_rows = [&](int tile) __attribute__((always_inline)) {
    int row = 256 * tile + 32 * w + l32;
    row = row < g.rows ? row : g.rows - 1;             // (what a row past the end gives is not stored)
    const uint8_t* const at = g.x + (int64_t)row * PITCH + 32 * hh;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      struct { uint4v a, b; } both = {*(const uint4v*)(at + 64 * s), *(const uint4v*)(at + 64 * s + 16)};
      xf[s] = __builtin_bit_cast(intx8, both);
    }
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) xe[i] = *(const int*)(g.xe + ((int64_t)i * g.rows + row) * 4);
    // (waited for here: left to their first use, the waits would stand in the loop and be for every younger load and store in each round)
#pragma unroll
    for (int s = 0; s < NS; ++s) asm volatile("" : "+v"(xf[s]));
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) asm volatile("" : "+v"(xe[i]));
  };

  // ---- ADD: what is added is where a column block's sum begins, four columns of a lane's row at a time, a step ahead.  (Rows past the
  // end: a buffer's loads past its last byte are zeros, its stores nothing, and all of them count.)
  typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
  uint2v cv[4];
  const uint32_t c_at = ADD ? (uint32_t)((32 * w + l32) * (int)g.c_stride + 4 * hh) * 2u : 0u;
  auto bytes_of = [&](int tile, int64_t stride, int from) __attribute__((always_inline)) {
    const int rows = g.rows - 256 * tile < 256 ? g.rows - 256 * tile : 256;
    return (int)(((int64_t)(rows - 1) * stride + (g.cols - from)) * 2);
  };
  auto ask_added = [&](int tile, int from) __attribute__((always_inline)) {
    const bf16_t* const base = (const bf16_t*)g.c + (int64_t)256 * tile * g.c_stride + from;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)scalar_ptr((const uint8_t*)base), 0, bytes_of(tile, g.c_stride, from), 0x00020000);
#pragma unroll
    for (int q = 0; q < 4; ++q) cv[q] = __builtin_amdgcn_raw_buffer_load_b64(r, (int)c_at + 16 * q, 0, 0);
  };
  auto added_here = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) asm volatile("" : "+v"(cv[q]));
  };

  // ---- the epilogue: 32 rows x 64 columns through the wave's own LDS in bf16, rows of 128 bytes, 8-byte piece c of row r at
  // c ^ (r / 2 % 16) (written a column piece of all rows at a time, read a row at a time: all banks both ways)
  uint8_t* const out_lds = smem + STAGES * STAGE + w * 4096;
  const int wslot = (l32 >> 1) & 15;
  floatx16 acc[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[1][i] = 0.f;        // (finished once before there is anything in it: into LDS, and not stored)
  // part `q4` of 4 of a column block: four columns of a lane's row
  auto finish = [&](auto par_, auto q_) __attribute__((always_inline)) {
    constexpr int par = decltype(par_)::value, q4 = decltype(q_)::value;
    float z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = acc[par][4 * q4 + i];
    if constexpr (OUT & ROWS_SILU) {
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = silu(z[i]);
    }
    *(uint2*)(out_lds + l32 * 128 + (((8 * par + 2 * q4 + hh) ^ wslot) * 8)) = uint2{pack2(z[0], z[1]), pack2(z[2], z[3])};
  };
  const bool halves = (lane >> 4) & 1;                 // (of 16 bytes, in the other order)
  const uint32_t out_at = (uint32_t)((32 * w + (lane >> 3)) * (int)g.out_stride + 8 * (lane & 7)) * 2u;
  const uint32_t out_step = 16u * (uint32_t)g.out_stride;
  const uint8_t* to_out = (const uint8_t*)g.out;       // where the pair in LDS goes
  int to_bytes = 0;
  auto store = [&]() __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)scalar_ptr(to_out), 0, to_bytes, 0x00020000);
    uint4v u[STORES];
#pragma unroll
    for (int i = 0; i < STORES; ++i) {
      const int row = (lane >> 3) + 8 * i;
      const uint4v v = *(const uint4v*)(out_lds + row * 128 + (((lane & 7) ^ ((row >> 2) & 7)) * 16));
      u[i] = uint4v{halves ? v[2] : v[0], halves ? v[3] : v[1], halves ? v[0] : v[2], halves ? v[1] : v[3]};
    }
#pragma unroll
    for (int i = 0; i < STORES; ++i) __builtin_amdgcn_raw_buffer_store_b128(u[i], r, (int)(out_at + i * out_step), 0, 2);
  };

  // ---- the run
#pragma unroll
  for (int t = 0; t < STAGES; ++t)
    if (left > 0) load_stage(t);
  load_rows(rt);
  if constexpr (ADD) {
    ask_added(rt, 64 * pc);
    added_here();
  }
  ROWS8_WAIT_VMCNT(0);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  int st = 0;
  exponents(0, 0);
  each<AHEAD>([&](auto s) __attribute__((always_inline)) { ask(0, s); });
  // One step: the products of a column block, the epilogue of the one before it, the stage after the next two on its way; in a pair's second
  // step the rows of the pair before are stored.
  auto step = [&](auto par_) __attribute__((always_inline)) {
    constexpr int par = decltype(par_)::value;
    const int next = st + 1 == STAGES ? 0 : st + 1;
    floatx16 begin;
#pragma unroll
    for (int i = 0; i < 16; ++i) begin[i] = !ADD ? 0.f : __builtin_bit_cast(float, i % 2 ? cv[i / 4][i % 4 / 2] & 0xffff0000u : cv[i / 4][i % 4 / 2] << 16);
    if constexpr (ADD) {
      const bool turn = par == 1 && pc + 1 == pairs;
      ask_added(turn ? (todo > 1 ? rt + 1 : rt) : rt, turn ? 0 : 64 * pc + (par == 0 ? 32 : 64));
    }
    if constexpr (par == 1) {
      store();
      to_out = (const uint8_t*)((const bf16_t*)g.out + (int64_t)256 * rt * g.out_stride + 64 * pc);
      to_bytes = bytes_of(rt, g.out_stride, 64 * pc);
    }
    each<NS>([&](auto s_) __attribute__((always_inline)) {
      constexpr int s = decltype(s_)::value, kb = s / 2;
      if constexpr (s + AHEAD < NS) {
        ask(st, std::integral_constant<int, s + AHEAD>{});
      } else {
        if constexpr (s + AHEAD == NS) {
          // everyone's last read of this stage is done, the next stage is here, and this one's place can be filled again.  Younger than the
          // next stage's loads: those of the one after it, and one pair's stores (in this step or the one before).
          if constexpr (ADD) added_here();
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (left > 0) ROWS8_WAIT_VMCNT(NLOAD + STORES);
          else ROWS8_WAIT_VMCNT(0);
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          if (left > 0) load_stage(st);
          exponents(next, par ^ 1);
        }
        ask(next, std::integral_constant<int, s + AHEAD - NS>{});
      }
      __builtin_amdgcn_sched_barrier(0);
      acc[par] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(f[s % (AHEAD + 1)], xf[s], s == 0 ? begin : acc[par], 0, 0, kb % 4, we[par][kb / 4], kb % 4, xe[kb / 4]);
      // the block before this one, a share of it behind each product
      each<4>([&](auto q) __attribute__((always_inline)) {
        if constexpr (decltype(q)::value * NS / 4 == s) finish(std::integral_constant<int, par ^ 1>{}, q);
      });
      asm volatile("" : "+v"(acc[par]));               // (the product stays here: the compiler would move it to where its result is used)
      __builtin_amdgcn_sched_barrier(0);
    });
    st = next;
  };
  while (true) {
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    if (--todo == 0) break;
    if (++pc == pairs) {
      pc = 0;
      load_rows(++rt);
    }
  }
  each<4>([&](auto q) __attribute__((always_inline)) { finish(std::integral_constant<int, 1>{}, q); });
  store();
}

// The products of up to 16 MT rows: a step of serving, where a call is a chain of latencies.  A workgroup takes 16 output columns and its
// waves one block of the contraction each in turn, straight from memory into their registers; their sums are added in LDS in the waves'
// order.  1 x 1024 to 4096 3.0 us (in tiles of 64 x 64, whose stages follow each other, 4.7), 1 x 8192 to 8192 14 us (4.6 TB/s).
constexpr int FEW_WAVES = 8;
template <int MT, bool F32>
__global__ __launch_bounds__(64 * FEW_WAVES) void hstu_rows8_few_kernel(const GemmParams g) {
  __shared__ floatx4 sums[FEW_WAVES][MT][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int l16 = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t pitch = (int64_t)g.blocks * BLOCK;
  // (rows past an operand's end are its last one: what they give is not stored)
  const int n = n0 + l16 < g.cols ? n0 + l16 : g.cols - 1;
  const uint8_t* const wr = g.w + n * pitch + 32 * q;
  const uint8_t* xr[MT];
  int m[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    m[t] = 16 * t + l16 < g.rows ? 16 * t + l16 : g.rows - 1;
    xr[t] = g.x + m[t] * pitch + 32 * q;
  }
  floatx4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = floatx4{0.f, 0.f, 0.f, 0.f};
  auto codes_of = [&](const uint8_t* at) __attribute__((always_inline)) {
    struct { uint4v a, b; } both = {*(const uint4v*)at, *(const uint4v*)(at + 16)};
    return __builtin_bit_cast(intx8, both);
  };
#pragma unroll 2
  for (int kb = w; kb < g.blocks; kb += waves) {
    const intx8 wf = codes_of(wr + kb * BLOCK);
    const int ws = g.we[((int64_t)(kb >> 2) * g.cols + n) * 4 + (kb & 3)];
    intx8 xf[MT];
    int xs[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      xf[t] = codes_of(xr[t] + kb * BLOCK);
      xs[t] = g.xe[((int64_t)(kb >> 2) * g.rows + m[t]) * 4 + (kb & 3)];
    }
    if constexpr (F32) {
      const float wp = power_of((uint32_t)ws);
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(values8(wf, i, wp), values8(xf[t], i, power_of((uint32_t)xs[t])), acc[t], 0, 0, 0);
    } else {
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf[t], acc[t], 0, 0, 0, ws, 0, xs[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) sums[w][t][lane] = acc[t];
  __syncthreads();
  for (int t = w; t < MT; t += waves) {
    floatx4 y = sums[0][t][lane];
    for (int i = 1; i < waves; ++i) {
      const floatx4 v = sums[i][t][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += v[e];
    }
    // the lane's four columns of row 16 t + l16
    const int row = 16 * t + l16, at = n0 + 4 * q;
    if (row >= g.rows || at >= g.cols) continue;
    if (g.c) add4<F32>(g.c, (int64_t)row * g.c_stride, at, g.cols, y);
    if (g.bias) add4<F32>(g.bias, 0, at, g.cols, y);
    if (g.activation) {
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = silu(y[e]);
    }
    if (at + 4 <= g.cols) {
      if constexpr (F32) *(floats4*)((float*)g.out + (int64_t)row * g.out_stride + at) = y;
      else *(words2*)((bf16_t*)g.out + (int64_t)row * g.out_stride + at) = words2{pack2(y[0], y[1]), pack2(y[2], y[3])};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (at + e < g.cols) {
          if constexpr (F32) ((float*)g.out)[(int64_t)row * g.out_stride + at + e] = y[e];
          else ((bf16_t*)g.out)[(int64_t)row * g.out_stride + at + e] = (bf16_t)y[e];
        }
    }
  }
}

// Raises a kernel's limit of dynamic LDS, once per device.
int allow_lds(const void* fn, int bytes, int* granted) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return rows8_fail(HSTU_ROWS8_ERR_LAUNCH, "no current device");
  if (dev >= 0 && dev < 64 && __atomic_load_n(&granted[dev], __ATOMIC_ACQUIRE) >= bytes) return HSTU_ROWS8_OK;
  const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return rows8_fail(HSTU_ROWS8_ERR_LAUNCH, "%d bytes of LDS: %s", bytes, hipGetErrorString(e));
  if (dev >= 0 && dev < 64) __atomic_store_n(&granted[dev], bytes, __ATOMIC_RELEASE);
  return HSTU_ROWS8_OK;
}

template <int MB, int NB, int WM, int WN, int STAGES, int KS, bool F32>
int launch_tiles(GemmParams g, hipStream_t st) {
  constexpr int TM = 32 * MB * WM, TN = 32 * NB * WN, LDS = lds_bytes(MB, NB, WM, WN, STAGES, KS);
  static_assert(LDS <= 160 << 10, "LDS");
  static int granted[64];
  const int64_t rt = ((int64_t)g.rows + TM - 1) / TM, ct = ((int64_t)g.cols + TN - 1) / TN;
  if (rt * ct > 0x7fffffffll / 16 || (rt * ct + 7) / 8 * 8 * 64 * WM * WN * KS > ROWS8_THREADS)
    return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "%d x %d outputs are too many for one call", g.rows, g.cols);
  g.row_tiles = (int32_t)rt;
  g.col_tiles = (int32_t)ct;
  const void* const fn = (const void*)hstu_rows8_gemm_kernel<MB, NB, WM, WN, STAGES, KS, F32>;
  if (const int rc = allow_lds(fn, LDS, granted)) return rc;
  hstu_rows8_gemm_kernel<MB, NB, WM, WN, STAGES, KS, F32><<<(uint32_t)((rt * ct + 7) / 8 * 8), 64 * WM * WN * KS, LDS, st>>>(g);
  return rows8_launched("hstu_rows8_gemm");
}

int launch_turns(GemmParams g, hipStream_t st) {
  constexpr int LDS = 2 * stage_bytes(256, 256);
  static int granted[64];
  const int64_t rt = ((int64_t)g.rows + 255) / 256, ct = ((int64_t)g.cols + 255) / 256;
  if ((rt * ct + 7) / 8 * 8 * 512 > ROWS8_THREADS) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "%d x %d outputs are too many for one call", g.rows, g.cols);
  g.row_tiles = (int32_t)rt;
  g.col_tiles = (int32_t)ct;
  if (const int rc = allow_lds((const void*)hstu_rows8_turns_kernel, LDS, granted)) return rc;
  hstu_rows8_turns_kernel<<<(uint32_t)((rt * ct + 7) / 8 * 8), 512, LDS, st>>>(g);
  return rows8_launched("hstu_rows8_gemm");
}

template <int MT, bool F32>
int launch_few(const GemmParams& g, hipStream_t st) {
  const int waves = g.blocks < FEW_WAVES ? g.blocks : FEW_WAVES;
  const int64_t groups = ((int64_t)g.cols + 15) / 16;
  if (groups * 64 * waves > ROWS8_THREADS) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "%d x %d outputs are too many for one call", g.rows, g.cols);
  hstu_rows8_few_kernel<MT, F32><<<(uint32_t)groups, 64 * waves, 0, st>>>(g);
  return rows8_launched("hstu_rows8_gemm");
}

template <int KB, int OUT>
int launch_rows(GemmParams g, hipStream_t st) {
  constexpr int LDS = 3 * (32 * KB * BLOCK + 256) + 8 * 4096;
  static int granted[64];
  const void* const fn = (const void*)hstu_rows8_rows_kernel<KB, OUT>;
  if (const int rc = allow_lds(fn, LDS, granted)) return rc;
  g.row_tiles = (g.rows + 255) / 256;
  hstu_rows8_rows_kernel<KB, OUT><<<256, 512, LDS, st>>>(g);
  return rows8_launched("hstu_rows8_gemm");
}

template <int OUT>
int launch_rows(const GemmParams& g, hipStream_t st) {
  switch (g.blocks) {
    case 1: return launch_rows<1, OUT>(g, st);
    case 2: return launch_rows<2, OUT>(g, st);
    case 3: return launch_rows<3, OUT>(g, st);
    case 4: return launch_rows<4, OUT>(g, st);
    case 5: return launch_rows<5, OUT>(g, st);
    case 6: return launch_rows<6, OUT>(g, st);
    case 7: return launch_rows<7, OUT>(g, st);
    default: return launch_rows<8, OUT>(g, st);
  }
}

// Whether the weight goes by rows kept in registers: bf16 results of contractions of up to 1024, whole pieces of 64 columns on whole vectors (else its
// stores, which go past the caches, are 280 us for 104 at 73728 x 512 to 2047, and through them no quicker than tiles), at least three
// pieces for each of the 256 workgroups (two: 4000 x 512 to 2048 12 us either way, 8000 x 512 to 2048, four of them, 16 against 19 in
// tiles) or, where rows are added, five (16398 x 1024 to 1024, four of them, 37 and in tiles 33; 32768 x 768 to 768, six, 33 and 38), and a quarter
// of the last rows' tile wasted at most.  Of rows to be added and a bias it takes one (a bias as rows without a stride).
bool rows_take(const GemmParams& g) {
  const int64_t tiles = ((int64_t)g.rows + 255) / 256, pieces = tiles * (g.cols / 64);
  return g.blocks <= 8 && g.cols % 64 == 0 && g.vec && !(g.c && g.bias) && pieces >= (g.c ? 1280 : 768) && 4 * (int64_t)g.rows >= 3 * 256 * tiles &&
         g.out_stride < 1 << 21 && g.c_stride < 1 << 21 && g.cols < 1 << 29;
}

// Up to 16 rows, or 32 where the weight is a small one, are latencies: 16 x 1024 to 4096 3.4 us, in tiles 4.8; 32 of them 3.7.  They are not where
// a great many columns of a short contraction read their rows of x anew every 16 columns: 8 x 512 to 100000 13.1 us, in tiles 10.9;
// 20000 columns 3.8 and 4.3, 1 x 8192 to 8192 14 and 20.
int few_take(const GemmParams& g) {
  if (g.rows <= 16 && (g.cols <= 32768 || g.blocks >= 16)) return 1;
  return g.rows <= 32 && g.cols <= 8192 && g.blocks <= 16 ? 2 : 0;
}

template <bool F32>
int launch(const GemmParams& g, hipStream_t st) {
  if (const int few = few_take(g)) return few == 1 ? launch_few<1, F32>(g, st) : launch_few<2, F32>(g, st);
  if constexpr (!F32) {
    if (rows_take(g)) {
      GemmParams r = g;
      if (g.bias) {
        r.c = g.bias;
        r.c_stride = 0;
      }
      return r.c ? (g.activation ? launch_rows<ROWS_ADD | ROWS_SILU>(r, st) : launch_rows<ROWS_ADD>(r, st))
                 : (g.activation ? launch_rows<ROWS_SILU>(r, st) : launch_rows<ROWS_PLAIN>(r, st));
    }
  }
  // The tiles under which the call is shortest, by what they were measured to take (us; b: blocks of the contraction, n: tiles to a CU).
  // Where tiles are one to a CU, sets of waves that share a long contraction out are what hides its latencies: 64 x 8192 to 8192 in tiles of 64
  // x 64 31 us, with four sets 19; 64 x 4096 to 16384 18 and 15; 400 x 1024 to 4096 6.2 and 9.0; in tiles of 128 x 128 800 x 4096 to 4096
  // 24 and with two sets 21, 400 x 8192 to 8192 45 and 36.
  //   64 x 64                 rounds of 4 to a CU, and for each block 0.2 a tile of a CU, or its latency
  //   64 x 64, four sets      n (3 + 0.21 b), less what operands that come from memory cost tiles that wait for them more often (64 x 1024 to 4096 among
  //                           a block's other steps 6.4 us without sets, 5.6 with; called over and over 4.6 and 4.7)
  //   128 x 128               rounds of two to a CU 4.2 + 0.9 b, of one 2.5 + 0.64 b
  //   128 x 128, two sets     n (4 + 0.52 b)
  //   256 x 256               9.3 + 1.46 b for a chip full of them, which its power sets; where the last round is not full, the clock is higher
  //                           (6000 x 4096 to 4096, a round and a half, 94 us; 16384 x 1024 to 1024, one, 22, and with 14 rows more 45)
  const float b = (float)g.blocks;
  auto tiles = [&](int64_t t) { return (((int64_t)g.rows + t - 1) / t) * (((int64_t)g.cols + t - 1) / t); };
  auto per = [&](int64_t t, int64_t chip) { return (float)((tiles(t) + chip - 1) / chip); };
  const float n64 = per(64, 256), n128 = per(128, 256), n256 = per(256, 256), step64 = F32 ? 0.277f * n64 : 0.2f * n64, latency = F32 ? 0.5f : 0.25f;
  const float one = F32 ? 3.f + 1.08f * b : 2.5f + 0.64f * b, two = F32 ? 6.1f + 1.7f * b : 4.2f + 0.9f * b;
  const int64_t rest = tiles(128) % 512;
  const float steps256 = F32 ? 3.0f * b * n256 : 1.46f * b * (float)tiles(256) / 256.f, least256 = F32 ? 0.f : 1.15f * b * n256;
  const float us[5] = {(F32 ? 2.9f : 2.0f) * per(64, 1024) + b * (step64 > latency ? step64 : latency),
                       n64 * ((F32 ? 3.8f : 3.f) + (F32 ? 0.29f : 0.21f) * b) - 0.8f,
                       (float)(tiles(128) / 512) * two + (rest > 256 ? two : rest ? one : 0.f),
                       n128 * ((F32 ? 6.f : 4.f) + (F32 ? 0.94f : 0.52f) * b),
                       n256 * (F32 ? 13.3f : 9.3f) + (steps256 > least256 ? steps256 : least256)};
  int best = 0;
  for (int i = 1; i < 5; ++i)
    if (us[i] < us[best]) best = i;
  switch (best) {
    case 0: return launch_tiles<1, 1, 2, 2, 2, 1, F32>(g, st);
    case 1: return launch_tiles<1, 1, 2, 2, 2, 4, F32>(g, st);
    case 2:
      // (eight waves of 32 x 64 rather than four of 64 x 64: 16398 x 1024 to 1024 with a residual 33 us for 37, 3000 x 1024 to 4096 19 for 22, 2000 x 512 to
      // 2048 6.8 for 7.4, 6000 x 4096 to 4096 97 for 94; in fp32, where a wave turns its codes into values, 184 for 191 the other way)
      if constexpr (F32) return launch_tiles<2, 2, 2, 2, 2, 1, true>(g, st);
      else return launch_tiles<1, 2, 4, 2, 2, 1, false>(g, st);
    case 3: return launch_tiles<2, 2, 2, 2, 2, 2, F32>(g, st);
    default:
      if constexpr (F32) return launch_tiles<4, 2, 2, 4, 2, 1, true>(g, st);
      else return launch_turns(g, st);
  }
}

int gemm(const HstuRows8GemmArgs* a, void* stream) {
  rows8_clear_error();
  if (!a) return rows8_fail(HSTU_ROWS8_ERR_NULL, "args is null");
  if (a->struct_size != sizeof(HstuRows8GemmArgs) || a->version != HSTU_ROWS8_ABI_VERSION)
    return rows8_fail(HSTU_ROWS8_ERR_VERSION, "struct_size %u version %u, expected %zu and %d", a->struct_size, a->version, sizeof(HstuRows8GemmArgs), HSTU_ROWS8_ABI_VERSION);
  if (const int rc = rows8_check(a->x, "x")) return rc;
  if (const int rc = rows8_check(a->w, "w")) return rc;
  if (a->x.width != a->w.width) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "x has rows of %d, w of %d", a->x.width, a->w.width);
  if (a->dtype != HSTU_ROWS8_BF16 && a->dtype != HSTU_ROWS8_FP32) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "dtype %d", a->dtype);
  if (a->activation != 0 && a->activation != 1) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "activation %d", a->activation);
  if (a->x.rows == 0 || a->w.rows == 0) return HSTU_ROWS8_OK;
  if (!a->out) return rows8_fail(HSTU_ROWS8_ERR_NULL, "out is null");
  const bool f32 = a->dtype == HSTU_ROWS8_FP32;
  for (const void* t : {(const void*)a->out, a->c, a->bias})
    if (t && ((uintptr_t)t & (f32 ? 3u : 1u))) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "a pointer is not aligned to its type");
  if (a->x.rows > 0x7fffffff - 256 || a->w.rows > 0x7fffffff - 256) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "%lld x %lld outputs are too many for one call", (long long)a->x.rows, (long long)a->w.rows);
  const int unit = f32 ? 4 : 8;
  GemmParams g = {};
  g.x = (const uint8_t*)a->x.codes; g.w = (const uint8_t*)a->w.codes;
  g.xe = (const uint8_t*)a->x.exponents; g.we = (const uint8_t*)a->w.exponents;
  g.out = a->out; g.c = a->c; g.bias = a->bias;
  g.out_stride = a->out_stride; g.c_stride = a->c_stride;
  g.rows = (int32_t)a->x.rows; g.cols = (int32_t)a->w.rows; g.blocks = rows8_blocks(a->x.width);
  g.activation = a->activation;
  g.vec = g.cols % 8 == 0 && rows8_aligned16(a->out) && a->out_stride % unit == 0 &&
          (!a->c || (rows8_aligned16(a->c) && a->c_stride % unit == 0));
  return f32 ? launch<true>(g, (hipStream_t)stream) : launch<false>(g, (hipStream_t)stream);
}

}  // namespace

extern "C" int hstu_rows8_gemm(const HstuRows8GemmArgs* args, void* stream) { return gemm(args, stream); }
