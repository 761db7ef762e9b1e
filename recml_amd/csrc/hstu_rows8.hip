// Rows of activations and weights in 8 bits, for gfx950 (MI355X): see include/hstu_rows8.h.
//
//   hstu_rows8_norm   rows, normed or as they are -> codes and block exponents
//   hstu_rows8_read   codes and exponents -> rows
//
// Both are passes over memory: a row is read once, stays in registers through the sum, the statistics (the mean, then the squares about it),
// the gate and the blocks' maxima, and leaves as one byte a value.  131072 x 512 in bf16 as they are 34 us (5.9 TB/s), with a norm 48, added to
// others 81 (5.8 TB/s), with a gate 58; 16398 x 1024 with norm and gate 14; a million of 64 45: half of what it writes there are the zeros
// behind each row.  In fp32 65536 x 1024 as they are 59 us (5.7 TB/s), with a norm 69, with a gate 105 (5.8 TB/s).  One row is a chain of
// latencies, 2 us.  A norm alone is bounded by its vector instructions, all else by memory (a large copy runs at 5.0 TB/s); read back,
// 131072 x 512 take 31 us (6.6 TB/s).

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "hstu_rows8_common.h"

namespace {
thread_local char g_err[512] = "";
}

int rows8_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

void rows8_clear_error() { g_err[0] = 0; }

int rows8_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HSTU_ROWS8_OK : rows8_fail(HSTU_ROWS8_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

int rows8_check(const HstuRows8& r, const char* name) {
  if (r.rows < 0 || r.rows > 0x7fffffffll) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "%s: %lld rows", name, (long long)r.rows);
  if (r.width < 1 || r.width > HSTU_ROWS8_MAX_WIDTH) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "%s: width=%d: 1 to %d", name, r.width, HSTU_ROWS8_MAX_WIDTH);
  if (r.rows == 0) return HSTU_ROWS8_OK;
  if (!r.codes || !r.exponents) return rows8_fail(HSTU_ROWS8_ERR_NULL, "%s: codes or exponents are null", name);
  if (!rows8_aligned16(r.codes) || ((uintptr_t)r.exponents & 3u)) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "%s: codes start on a 16-byte boundary, exponents on a 4-byte one", name);
  return HSTU_ROWS8_OK;
}

namespace {

struct Params {
  const void *x, *add, *gate, *gamma, *beta;
  void* sum;
  uint8_t* codes;
  uint8_t* exponents;
  int64_t x_stride, add_stride, gate_stride, sum_stride;
  int64_t rows;
  int32_t width;
  float eps;
};

// Eight values of a row as they lie in memory, at any place that the type may have: the wide accesses of this chip need no more.
typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef float floats4 __attribute__((ext_vector_type(4), aligned(4)));
template <bool F32>
struct Eight {
  uint4v w[F32 ? 2 : 1];
};

// How rows go into pieces of 8: evenly, or with a last piece that is not whole, or into one that is not.
enum { FIT_EVEN, FIT_REST, FIT_PART };

// Eight values from column `col` on; past the width zeros.  No branch: a piece that is not whole is the row's last eight values, moved down.
// (Through the caches: past them rows of 268 MB are quicker, 65536 x 2048 as they are 71 -> 63 us, and those of 34 MB slower, 10.0 -> 11.4, as three
// operands are, 161 -> 172 and 20 -> 23.)
template <bool F32, int FIT>
__device__ __forceinline__ Eight<F32> load8(const void* base, int64_t at, int col, int width) {
  constexpr int N = F32 ? 8 : 4;                   // words
  Eight<F32> x = {};
  uint32_t w[N];
  if constexpr (FIT == FIT_PART) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = 0u;
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (col + i < width) {
        if constexpr (F32) w[i] = ((const uint32_t*)base)[at + col + i];
        else w[i / 2] |= (uint32_t)((const uint16_t*)base)[at + col + i] << (16 * (i % 2));
      }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) x.w[i] = uint4v{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
    return x;
  }
  const int from = col < width - 8 ? col : width - 8, down = col - from;
  if constexpr (F32) {
    const floats4* const p = (const floats4*)((const float*)base + at + from);
    x.w[0] = __builtin_bit_cast(uint4v, (floatx4)p[0]);
    x.w[1] = __builtin_bit_cast(uint4v, (floatx4)p[1]);
  } else {
    x.w[0] = *(const words4*)((const bf16_t*)base + at + from);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = x.w[i / 4][i % 4];
  if constexpr (FIT == FIT_REST) {
    auto move = [&](int words, bool on) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t v = i + words < N ? w[i + words < N ? i + words : 0] : 0u;
        w[i] = on ? v : w[i];
      }
    };
    if constexpr (!F32) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t v = __builtin_amdgcn_alignbit(i + 1 < N ? w[i + 1 < N ? i + 1 : 0] : 0u, w[i], 16);
        w[i] = down & 1 ? v : w[i];
      }
      move(1, down & 2);
      move(2, down & 4);
    } else {
      move(1, down & 1);
      move(2, down & 2);
      move(4, down & 4);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = down < 8 ? w[i] : 0u;
#pragma unroll
  for (int i = 0; i < N / 4; ++i) x.w[i] = uint4v{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
  return x;
}
template <bool F32>
__device__ __forceinline__ void values_of(const Eight<F32>& x, float (&f)[8]) {
  if constexpr (F32) {
    const floatx4 lo = __builtin_bit_cast(floatx4, x.w[0]), hi = __builtin_bit_cast(floatx4, x.w[1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = lo[i]; f[4 + i] = hi[i]; }
  } else {
    unpack8(x.w[0], f);
  }
}

template <bool F32>
__device__ __forceinline__ void store8(void* base, int64_t at, int col, int width, const float (&f)[8]) {
  if (col + 8 <= width) {
    if constexpr (F32) {
      floats4* const to = (floats4*)((float*)base + at + col);
      to[0] = floats4{f[0], f[1], f[2], f[3]};
      to[1] = floats4{f[4], f[5], f[6], f[7]};
    } else {
      *(words4*)((bf16_t*)base + at + col) = pack8(f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (col + i < width) {
        if constexpr (F32) ((float*)base)[at + col + i] = f[i];
        else ((bf16_t*)base)[at + col + i] = (bf16_t)f[i];
      }
  }
}

// a value of the lane's neighbour in a row of 16: quad_perm [1,0,3,2] and [2,3,0,1], row_half_mirror, row_mirror
template <int CTRL>
__device__ __forceinline__ uint32_t of_neighbour(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true); }
template <int CTRL>
__device__ __forceinline__ float add_neighbour(float v) { return v + __builtin_bit_cast(float, of_neighbour<CTRL>(__builtin_bit_cast(uint32_t, v))); }
template <int CTRL>
__device__ __forceinline__ double add_neighbour(double v) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  return v + __builtin_bit_cast(double, (uint64_t)of_neighbour<CTRL>((uint32_t)(w >> 32)) << 32 | of_neighbour<CTRL>((uint32_t)w));
}
template <int CTRL>
__device__ __forceinline__ uint32_t max_neighbour(uint32_t v) {
  const uint32_t o = of_neighbour<CTRL>(v);
  return o > v ? o : v;
}
// the largest of a block's 16 threads (of fewer where a row has no more)
template <int T>
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
  v = max_neighbour<0xB1>(v);
  if constexpr (T >= 4) v = max_neighbour<0x4E>(v);
  if constexpr (T >= 8) v = max_neighbour<0x141>(v);
  if constexpr (T >= 16) v = max_neighbour<0x140>(v);
  return v;
}

// the sum over a row's T threads, the same bits in each of them
template <int T, class Y>
__device__ __forceinline__ Y row_sum(Y v, Y* parts) {
  v = add_neighbour<0xB1>(v);
  if constexpr (T >= 4) v = add_neighbour<0x4E>(v);
  if constexpr (T >= 8) v = add_neighbour<0x141>(v);
  if constexpr (T >= 16) v = add_neighbour<0x140>(v);
  if constexpr (T >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (T >= 64) v += __shfl_xor(v, 32, 64);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) v += parts[w];
    __syncthreads();
  }
  return v;
}

// What a row's values are until they become codes.  Rows in 32 bits take 64: a value next to a border between two codes takes the one that it has by
// the definition, where in fp32 5e-7 of them take the other, a whole 2^-3 away, and a block's steps in a row come out 1e-4 off instead of 3e-8.
// A norm alone pays for it, 65536 x 1024 69 us for 58, 16384 x 999 25 for 17; with a gate 105 for 107.  (Rows in bf16 are no nearer to what they
// stand for than 2^-9; theirs is fp32, in which 5e-7 of the codes are the neighbour.)
template <bool F32> struct ValueOf { typedef float type; };
template <> struct ValueOf<true> { typedef double type; };

// As fp32, of a value in 64 bits its first 20 with what comes behind them in the last one (set where any of it is), so that the rounding
// to a code of 4, and the comparison with a border, are those of the value.
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(double v) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)w;
  return (float)__builtin_bit_cast(double, (uint64_t)((uint32_t)(w >> 32) | (lo < 1u ? lo : 1u)) << 32);
}
__device__ __forceinline__ float inverse_root(float v) { return __builtin_amdgcn_rsqf(v); }
// (squares past fp32 are infinite ones for rows of either type)
__device__ __forceinline__ double inverse_root(double v) { return v > 0x1.fffffep127 ? 0. : 1. / sqrt(v); }

constexpr int threads_of(int t) { return t < 256 ? 256 : t; }

// T threads a row (2 of 16 values up to a workgroup), V pieces of 8 values each: piece v of thread t holds the values from 8 (v T + t) on, so a block's are 16 neighbours.
// Everything that a row needs is asked for at once: gamma, beta and gate behind the statistics would be a second latency (but for the widest rows
// in 32 bits, which have no registers for it: 2048 x 32768 with a gate 139 us for 310).  MORE: there is
// something to add or a gate; what is not there (nor beta) is read from x (gamma) once more and left out, so that no branch parts the loads.
template <bool F32, int NORM, bool MORE, int FIT, int T, int V>
__global__ __launch_bounds__(threads_of(T)) void hstu_rows8_norm_kernel(const Params p) {
  using Y = typename ValueOf<F32>::type;
  __shared__ Y parts[T > 64 ? T / 64 : 1];
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * (threads_of(T) / T) + threadIdx.x / T;
  if (row >= p.rows) return;                       // (T > 64: a row is the whole workgroup)
  const int W = p.width, blocks = rows8_blocks(W);
  constexpr bool LATE = F32 && V > 2;               // (registers for what follows the statistics only then)
  Eight<F32> x[V], added[V], gate[V], gamma[V], beta[V];
  auto affine = [&](int v) __attribute__((always_inline)) {
    const int col = 8 * (v * T + t);
    if constexpr (MORE) gate[v] = load8<F32, FIT>(p.gate ? p.gate : p.x, row * (p.gate ? p.gate_stride : p.x_stride), col, W);
    if constexpr (NORM != HSTU_ROWS8_AS_IS) {
      gamma[v] = load8<F32, FIT>(p.gamma, 0, col, W);
      beta[v] = load8<F32, FIT>(p.beta ? p.beta : p.gamma, 0, col, W);
    }
  };
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int col = 8 * (v * T + t);
    x[v] = load8<F32, FIT>(p.x, row * p.x_stride, col, W);
    if constexpr (MORE) added[v] = load8<F32, FIT>(p.add ? p.add : p.x, row * (p.add ? p.add_stride : p.x_stride), col, W);
    if constexpr (!LATE) affine(v);
  }
  float f[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) values_of<F32>(x[v], f[v]);
  if (MORE && p.add) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a[8];
      values_of<F32>(added[v], a);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[v][i] += a[i];
        if constexpr (!F32) f[v][i] = (float)(bf16_t)f[v][i];
      }
      if (p.sum) store8<F32>(p.sum, row * p.sum_stride, 8 * (v * T + t), W, f[v]);
    }
  }
  Y mean = 0, rstd = 1;
  // (past the width: values are zeros, and so are their differences; gamma and beta are zeros too)
  auto difference = [&](int v, int i) __attribute__((always_inline)) {
    if constexpr (NORM == HSTU_ROWS8_LAYER) return (Y)f[v][i] - (8 * (v * T + t) + (FIT == FIT_EVEN ? 0 : i) < W ? mean : (Y)0);
    else return (Y)f[v][i];
  };
  if constexpr (NORM != HSTU_ROWS8_AS_IS) {
    // (divided, not multiplied by 1 / W: the mean of equal values is that value, and their differences from it are zeros)
    const Y count = (Y)W;
    if constexpr (NORM == HSTU_ROWS8_LAYER) {
      Y s[2] = {0, 0};
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i & 1] += f[v][i];
      mean = row_sum<T, Y>(s[0] + s[1], parts) / count;
    }
    Y ss[2] = {0, 0};
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const Y d = difference(v, i);
        ss[i & 1] = fma(d, d, ss[i & 1]);
      }
    rstd = inverse_root(row_sum<T, Y>(ss[0] + ss[1], parts) / count + (Y)p.eps);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if constexpr (LATE) affine(v);
    if constexpr (LATE) {                            // (the values stay in 32 bits: their differences are taken again)
#pragma unroll
      for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(f[v][i]));
    }
    Y y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = difference(v, i);
    if constexpr (NORM != HSTU_ROWS8_AS_IS) {
      float g[8];
      values_of<F32>(gamma[v], g);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = F32 ? y[i] * (rstd * g[i]) : y[i] * rstd * g[i];
      if (p.beta) {
        values_of<F32>(beta[v], g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma clang fp contract(off)      // (every step rounded, as it is in separate operations: half as many codes differ from theirs, 5e-7 of them)
          y[i] = y[i] + g[i];
        }
      }
    }
    if (MORE && p.gate) {
      float u[8];
      values_of<F32>(gate[v], u);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= u[i];
    }
    const int piece = v * T + t, block = piece / 16;
    uint32_t top = 0;
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      z[i] = as_float(y[i]);
      const uint32_t m = __builtin_bit_cast(uint32_t, z[i]) & 0x7fffffffu;
      top = m > top ? m : top;
    }
    top = block_max<T>(top);
    // floor(log2 top) less the largest code's 8, one more where top is past 464 = 1.8125 * 2^8 powers
    int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x680000u ? 1 : 0);
    e = e < 1 ? 1 : e > 246 ? 246 : e;              // (top = 0 too)
    const bool bad = top >= 0x7f800000u;
    const float inverse = power_of(254 - (uint32_t)e);
    uint2 code;
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = __builtin_amdgcn_fmed3f(z[i] * inverse, -448.f, 448.f);
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
    code.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], c, true);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(z[4], z[5], 0, false);
    code.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[6], z[7], c, true);
    uint8_t* const to = p.codes + row * ((int64_t)blocks * BLOCK) + 8 * piece;
    if (block < blocks) *(uint2*)to = bad ? uint2{0u, 0u} : code;
#pragma unroll
    for (int i = T; i < 16; i += T) *(uint2*)(to + 8 * i) = uint2{0u, 0u};
    if (t % 16 == 0 && block < (blocks + 3) / 4 * 4)
      p.exponents[((int64_t)(block / 4) * p.rows + row) * 4 + block % 4] = block >= blocks ? (uint8_t)1 : bad ? (uint8_t)255 : (uint8_t)e;
    // (groups whose last blocks no thread has)
    if (v == V - 1 && t == T - 1) {
      for (int more = block + 1; more < (blocks + 3) / 4 * 4; ++more) p.exponents[((int64_t)(more / 4) * p.rows + row) * 4 + more % 4] = 1;
    }
  }
}

struct ReadParams {
  const uint8_t* codes;
  const uint8_t* exponents;
  void* out;
  int64_t out_stride, rows;
  int32_t width;
  int32_t pieces;          // of 8 values, in a row
};

// a piece of 8 values a thread
template <bool F32>
__global__ __launch_bounds__(256) void hstu_rows8_read_kernel(const ReadParams p) {
  const uint32_t at = blockIdx.x * 256u + threadIdx.x, of = at / (uint32_t)p.pieces;      // (a launch has fewer than 2^32 threads)
  const int64_t row = of;
  const int piece = (int)(at - of * (uint32_t)p.pieces);
  if (row >= p.rows) return;
  const uint2 w = *(const uint2*)(p.codes + row * ((int64_t)rows8_blocks(p.width) * BLOCK) + 8 * piece);
  const int block = piece / 16;
  const uint32_t e = p.exponents[((int64_t)(block / 4) * p.rows + row) * 4 + block % 4];
  const float power = e == 255u ? __builtin_nanf("") : power_of(e);
  const floatx2 y[4] = {__builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false), __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true),
                        __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false), __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true)};
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = y[i / 2][i % 2] * power;
  store8<F32>(p.out, row * p.out_stride, 8 * piece, p.width, f);
}

template <bool F32, int NORM, bool MORE, int FIT, int T, int V>
int launch_norm(const Params& p, hipStream_t st) {
  constexpr int THREADS = threads_of(T), ROWS = THREADS / T;      // of a workgroup
  const int64_t groups = (p.rows + ROWS - 1) / ROWS;
  if (groups > ROWS8_THREADS / THREADS) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "%lld rows of %d are too many for one call", (long long)p.rows, p.width);
  hstu_rows8_norm_kernel<F32, NORM, MORE, FIT, T, V><<<(uint32_t)groups, THREADS, 0, st>>>(p);
  return rows8_launched("hstu_rows8_norm");
}

template <bool F32, int NORM, bool MORE, int FIT>
int launch_norm(const Params& p, hipStream_t st) {
  // (479394 x 9, normed, 45 us by eight threads a row, 31 by two; 302579 x 21 with a gate 24 and, by four, 18; as they are, where the zeros behind the values are most of the work, 250075 x 9 11 and 15)
  constexpr int FEW = NORM == HSTU_ROWS8_AS_IS ? 8 : 2, SOME = NORM == HSTU_ROWS8_AS_IS ? 8 : 4;
#define ROWS8_LAUNCH(T, V) return launch_norm<F32, NORM, MORE, FIT, T, V>(p, st)
  if constexpr (FIT == FIT_PART) {
    ROWS8_LAUNCH(FEW, 1);
  } else {
    if (p.width <= 8 * FEW) ROWS8_LAUNCH(FEW, 1);
    if (p.width <= 8 * SOME) ROWS8_LAUNCH(SOME, 1);
    if (p.width <= 64) ROWS8_LAUNCH(8, 1);
    if (p.width <= 128) ROWS8_LAUNCH(16, 1);
    if (p.width <= 256) ROWS8_LAUNCH(32, 1);
    if (p.width <= 512) ROWS8_LAUNCH(64, 1);
    if (p.width <= 1024) ROWS8_LAUNCH(64, 2);
    if constexpr (F32) {                           // (values in 64 bits leave registers for two pieces)
      if (p.width <= 2048) ROWS8_LAUNCH(64, 4);
      if (p.width <= 4096) ROWS8_LAUNCH(256, 2);
      if (p.width <= 8192) ROWS8_LAUNCH(256, 4);
      ROWS8_LAUNCH(1024, 4);
    } else {
      if (p.width <= 2048) ROWS8_LAUNCH(64, 4);
      if (p.width <= 8192) ROWS8_LAUNCH(256, 4);
      ROWS8_LAUNCH(1024, 4);
    }
  }
#undef ROWS8_LAUNCH
}

template <bool F32, int NORM, bool MORE>
int launch_norm(const Params& p, hipStream_t st) {
  if (p.width < 8) return launch_norm<F32, NORM, MORE, FIT_PART>(p, st);
  return p.width % 8 == 0 ? launch_norm<F32, NORM, MORE, FIT_EVEN>(p, st) : launch_norm<F32, NORM, MORE, FIT_REST>(p, st);
}

template <bool F32, int NORM>
int launch_norm(const Params& p, hipStream_t st) {
  if constexpr (NORM != HSTU_ROWS8_AS_IS) {
    if (p.add || p.gate) return launch_norm<F32, NORM, true>(p, st);
  }
  return launch_norm<F32, NORM, false>(p, st);
}

template <bool F32>
int launch_norm(const Params& p, int norm, hipStream_t st) {
  if (norm == HSTU_ROWS8_LAYER) return launch_norm<F32, HSTU_ROWS8_LAYER>(p, st);
  return norm == HSTU_ROWS8_RMS ? launch_norm<F32, HSTU_ROWS8_RMS>(p, st) : launch_norm<F32, HSTU_ROWS8_AS_IS>(p, st);
}

int norm_rows(const HstuRows8NormArgs* a, void* stream) {
  rows8_clear_error();
  if (!a) return rows8_fail(HSTU_ROWS8_ERR_NULL, "args is null");
  if (a->struct_size != sizeof(HstuRows8NormArgs) || a->version != HSTU_ROWS8_ABI_VERSION)
    return rows8_fail(HSTU_ROWS8_ERR_VERSION, "struct_size %u version %u, expected %zu and %d", a->struct_size, a->version, sizeof(HstuRows8NormArgs), HSTU_ROWS8_ABI_VERSION);
  if (const int rc = rows8_check(a->rows, "rows")) return rc;
  if (a->dtype != HSTU_ROWS8_BF16 && a->dtype != HSTU_ROWS8_FP32) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "dtype %d", a->dtype);
  if (a->norm < HSTU_ROWS8_AS_IS || a->norm > HSTU_ROWS8_RMS) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "norm %d", a->norm);
  if (a->sum && !a->add) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "a sum needs something to add");
  if (a->norm == HSTU_ROWS8_AS_IS && (a->add || a->gate)) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "rows as they are have nothing added and no gate");
  if (a->rows.rows == 0) return HSTU_ROWS8_OK;
  if (!a->x) return rows8_fail(HSTU_ROWS8_ERR_NULL, "x is null");
  if (a->norm != HSTU_ROWS8_AS_IS && !a->gamma) return rows8_fail(HSTU_ROWS8_ERR_NULL, "gamma is null");
  const bool f32 = a->dtype == HSTU_ROWS8_FP32;
  for (const void* t : {a->x, a->add, a->gate, (const void*)a->sum, a->gamma, a->beta})
    if ((uintptr_t)t & (f32 ? 3u : 1u)) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "a pointer is not aligned to its type");
  Params p;
  p.x = a->x; p.add = a->add; p.gate = a->gate; p.gamma = a->gamma; p.beta = a->beta; p.sum = a->sum;
  p.codes = (uint8_t*)a->rows.codes; p.exponents = (uint8_t*)a->rows.exponents;
  p.x_stride = a->x_stride; p.add_stride = a->add_stride; p.gate_stride = a->gate_stride; p.sum_stride = a->sum_stride;
  p.rows = a->rows.rows; p.width = a->rows.width; p.eps = a->eps;
  hipStream_t st = (hipStream_t)stream;
  return f32 ? launch_norm<true>(p, a->norm, st) : launch_norm<false>(p, a->norm, st);
}

int read_rows(const HstuRows8ReadArgs* a, void* stream) {
  rows8_clear_error();
  if (!a) return rows8_fail(HSTU_ROWS8_ERR_NULL, "args is null");
  if (a->struct_size != sizeof(HstuRows8ReadArgs) || a->version != HSTU_ROWS8_ABI_VERSION)
    return rows8_fail(HSTU_ROWS8_ERR_VERSION, "struct_size %u version %u, expected %zu and %d", a->struct_size, a->version, sizeof(HstuRows8ReadArgs), HSTU_ROWS8_ABI_VERSION);
  if (const int rc = rows8_check(a->rows, "rows")) return rc;
  if (a->dtype != HSTU_ROWS8_BF16 && a->dtype != HSTU_ROWS8_FP32) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "dtype %d", a->dtype);
  if (a->rows.rows == 0) return HSTU_ROWS8_OK;
  if (!a->out) return rows8_fail(HSTU_ROWS8_ERR_NULL, "out is null");
  const bool f32 = a->dtype == HSTU_ROWS8_FP32;
  if ((uintptr_t)a->out & (f32 ? 3u : 1u)) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "out is not aligned to its type");
  ReadParams p;
  p.codes = (const uint8_t*)a->rows.codes; p.exponents = (const uint8_t*)a->rows.exponents;
  p.out = a->out; p.out_stride = a->out_stride; p.rows = a->rows.rows; p.width = a->rows.width;
  p.pieces = (p.width + 7) / 8;
  const int64_t all = p.rows * p.pieces;
  if (all > ROWS8_THREADS - 256) return rows8_fail(HSTU_ROWS8_ERR_SHAPE, "%lld rows of %d are too many for one call", (long long)p.rows, p.width);
  const uint32_t grid = (uint32_t)((all + 255) / 256);
  hipStream_t st = (hipStream_t)stream;
  if (f32) hstu_rows8_read_kernel<true><<<grid, 256, 0, st>>>(p);
  else hstu_rows8_read_kernel<false><<<grid, 256, 0, st>>>(p);
  return rows8_launched("hstu_rows8_read");
}

}  // namespace

extern "C" {

int hstu_rows8_norm(const HstuRows8NormArgs* args, void* stream) { return norm_rows(args, stream); }
int hstu_rows8_read(const HstuRows8ReadArgs* args, void* stream) { return read_rows(args, stream); }
int hstu_rows8_abi_version(void) { return HSTU_ROWS8_ABI_VERSION; }
const char* hstu_rows8_last_error(void) { return g_err; }

}
