// Attention of new events over kept keys and values in 4 or 8 bits, for gfx950 (MI355X): see include/hstu_serve.h.
//
//   out_i = 1/n sum_{j <= i} silu(alpha q_i . k_j + pos[L - 1 + j - i] + ts_w[bucket(ts_{i + 1} - ts_j)]) v_j
//
// There is no softmax, so parts of the keys are independent sums: a workgroup takes `chunk` keys of one (sequence, head,
// block of queries), its four waves every fourth 32 of them, and where a sequence has several parts a second kernel adds
// them in order.
//
// A wave's step is 32 keys on the 16x16x32 bf16 matrix instruction.  Both formats are exact in bf16 (2 or 4 significant
// bits times a power of two), so codes become operands by the hardware's scaled conversions without rounding:
//   S^T = K Q^T   rows are keys.  Row r of tile t is key 8 (r / 4) + 4 t + r % 4, so that the lanes that get a query's
//                 logits hold eight consecutive keys of it: exactly the eight that the second product's operand wants
//                 of them, and the activated weights go from registers to registers.
//   O^T = V^T P^T rows are the head's dims.  A lane reads its own run of d / 16 dims of its eight keys, scales each key's
//                 run by that key's exponent on conversion, and pairs the keys up with byte permutes: nothing goes
//                 through LDS, and the cache keeps rows as they are written.
// The contraction order along d and along the keys is free as long as both operands agree: K's lane takes a run of d / 4
// dims (one block of exponents at d = 128), and Q is read the same way.
// Queries in fp32 run as three bf16 parts (24 bits: all of them); activated weights as two for bf16 results (2^-17 of a weight is
// lost, where one part would lose 2^-9 and make half of the result's error), as three for fp32 ones.
// Biases with timestamps are worked out by the whole workgroup, a pair a thread, for up to 8192 pairs ahead: done where the logits
// lie, a single query's would cost each wave 16 times the work, since its 16 columns hold one row.  Positions alone are the entries
// of the table that the block's places span, once.
//
// What bounds it (d = 128 in 4 bits, 8 heads, one query a sequence): long histories read the cache at memory's rate, 192 sequences of
// 4096 keys, 857 MB, in 157 us (5.5 TB/s; the vector pipes are busy for 56 % of that, mostly with scaling and pairing codes, which is why
// no step of it may wait).  Short and uneven ones take as long as the longest part's chain of dependent steps: 64 sequences of
// up to 2048 keys of power-law length, 18 MB, 14 us and the join 4; a single sequence of 2048 keys 7.5 and 4.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "hstu_serve_common.h"

namespace {

typedef __attribute__((address_space(4))) int32_t Constant;   // what no kernel writes while this one runs

constexpr int WAVES = 4;
constexpr int THREADS = 64 * WAVES;
constexpr int STEP = 32;             // keys of a wave's step
constexpr int MAX_BUCKETS = 128;
constexpr int BUCKET_FLOATS = 2 * MAX_BUCKETS + 4;   // the buckets' thresholds and values in LDS

struct Params {
  HstuKvPages g;
  const int32_t* lengths;
  const int32_t* offsets;
  const void* q;
  void* out;
  int64_t total;
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;
  const float* pos;
  const int64_t* ts;
  const float* ts_tab;
  float* partial;                    // [row][head][part][d], null with one part
  int32_t per_seq, max_len, pos_heads, ts_heads, ts_buckets;
  int32_t chunk, parts, qblocks, sub_log2;
  float alpha, inv_n, buckets_per_log2;
  int32_t thr[MAX_BUCKETS + 2];      // thr[b]: smallest time difference of bucket b or a later one
};

// What a sequence's geometry says of the call: its first row, its rows, the place of row 0, and how many places are there.
struct Seq {
  int64_t first, place0;
  int count, limit, last_ts;
};

__device__ __forceinline__ Seq seq_of(const Params& p, int b) {
  Seq s;
  if (p.offsets) {
    int64_t o0 = p.offsets[b], o1 = p.offsets[b + 1];
    o0 = o0 < 0 ? 0 : o0 > p.total ? p.total : o0;
    o1 = o1 < o0 ? o0 : o1 > p.total ? p.total : o1;
    s.first = o0;
    s.count = (int)(o1 - o0 < p.per_seq ? o1 - o0 : p.per_seq);
  } else {
    s.first = (int64_t)b * p.per_seq;
    s.count = p.per_seq;
  }
  const int n = p.lengths[b];
  s.place0 = (int64_t)n - s.count;
  const int64_t held = (int64_t)p.g.table_pages * p.g.page_size;
  int limit = n < p.max_len ? n : p.max_len;
  limit = limit < held ? limit : (int)held;
  if (p.g.n_pages == 0) limit = 0;
  s.limit = limit < 0 ? 0 : limit;
  s.last_ts = (n < p.max_len ? n : p.max_len) - 1;
  return s;
}

// One past the last key that row t attends to (0: none, its output is zeros).
__device__ __forceinline__ int keys_of(const Seq& s, int t) {
  const int64_t i = s.place0 + t;
  return t < s.count && i >= 0 && i < s.limit ? (int)i + 1 : 0;
}

template <int N>
struct Bytes { uint32_t w[N < 4 ? 1 : N / 4]; };

template <int N>
__device__ __forceinline__ Bytes<N> load_bytes(const uint8_t* at) {
  Bytes<N> r;
  if constexpr (N == 1) r.w[0] = *at;
  else if constexpr (N == 2) r.w[0] = *(const uint16_t*)at;
  else if constexpr (N == 4) r.w[0] = *(const uint32_t*)at;
  else if constexpr (N == 8) { const uint2 v = *(const uint2*)at; r.w[0] = v.x; r.w[1] = v.y; }
  else {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const uint4 v = ((const uint4*)at)[i];
      r.w[4 * i] = v.x; r.w[4 * i + 1] = v.y; r.w[4 * i + 2] = v.z; r.w[4 * i + 3] = v.w;
    }
  }
  return r;
}

// Values 2 I and 2 I + 1 of a run of codes, times `power`, as a pair of bf16.
template <int BITS, int I, int N>
__device__ __forceinline__ uint32_t pair_at(const Bytes<N>& c, float power) {
  if constexpr (BITS == 4) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.w[I / 4], power, I % 4));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.w[I / 2], power, I % 2 == 1));
}

template <int BITS, int N, int COUNT, int I = 0>
__device__ __forceinline__ void pairs_of(const Bytes<N>& c, float power, uint32_t* out) {
  if constexpr (I < COUNT) {
    out[I] = pair_at<BITS, I>(c, power);
    pairs_of<BITS, N, COUNT, I + 1>(c, power, out);
  }
}

template <int I, int N, typename F>
__device__ __forceinline__ void each_pair(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each_pair<I + 1, N>(f);
  }
}

__device__ __forceinline__ bf16x8 operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(bf16x8, uint4{a, b, c, d});
}

// x as bf16 parts whose sum it is (the third one takes what is left to its last bit).  KEEP: an infinity stays one (without, it becomes
// NaN: a weight past fp32, where the row's sum is not finite either way).
template <int PARTS, bool KEEP>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&out)[PARTS]) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
  for (int n = 0; n < PARTS; ++n) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack2(rest[2 * i], rest[2 * i + 1]);
      if (n + 1 < PARTS) {
        const float lo = __builtin_bit_cast(float, w[i] << 16), hi = __builtin_bit_cast(float, w[i] & 0xffff0000u);
        rest[2 * i] = KEEP && __builtin_isinf(lo) ? 0.f : rest[2 * i] - lo;
        rest[2 * i + 1] = KEEP && __builtin_isinf(hi) ? 0.f : rest[2 * i + 1] - hi;
      }
    }
    out[n] = operand(w[0], w[1], w[2], w[3]);
  }
}

// The buckets of time differences, in LDS: thr[b] the smallest difference of bucket b or a later one, tab[b] its value.
struct Buckets {
  const int32_t* thr;
  const float* tab;
  int32_t count;
  float per_log2;            // ln 2 over a bucket's size
};

__device__ __forceinline__ float bucket_value(const Buckets& t, int64_t gap) {
  gap = gap < 0 ? -gap : gap;
  const int dt = gap < 1 ? 1 : gap > 1000000000 ? 1000000000 : (int)gap;
  int b = (int)(__builtin_amdgcn_logf((float)dt) * t.per_log2);
  b = b < 0 ? 0 : b > t.count ? t.count : b;                // (off by one at most: its neighbours' borders decide)
  const int lo = t.thr[b], hi = t.thr[b + 1];
  b += (dt >= hi ? 1 : 0) - (dt < lo ? 1 : 0);
  return t.tab[b];
}

// Waves a SIMD that the registers are cut for.
constexpr int waves_of(int dp, bool f32, int nq) { return f32 || dp > 128 || nq == 4 ? 1 : nq == 1 || dp <= 64 ? 3 : 2; }

// What a wave's step reads of its 32 keys.
template <int DP, int BITS>
struct Raw {
  static constexpr int KB = DP / 4 * BITS / 8;       // bytes of a lane's run of a key
  static constexpr int KBLK = DP > 128 ? 2 : 1;      // blocks of exponents in it
  static constexpr int VN = DP / 16;                 // dims of a lane's run of a value
  static constexpr int VB = VN * BITS / 8;
  Bytes<KB> k[2];
  uint32_t ke[2][KBLK];
  Bytes<VB> v[8];
  uint32_t ve[2];
};

template <int DP, bool EXACT, int BITS, bool F32, int NQ>
__global__ __launch_bounds__(THREADS, waves_of(DP, F32, NQ)) void hstu_cached_attn_kernel(const Params p) {
  using R = Raw<DP, BITS>;
  constexpr int QP = F32 ? 3 : 1;             // bf16 parts of queries
  constexpr int WP = F32 ? 3 : 2;             // and of weights
  constexpr int KS = DP / 32;                 // matrix steps along d
  constexpr int VN = R::VN;
  constexpr int ACC = VN * 4 * NQ;            // accumulators of a lane
  // sums of two waves [2][ACC][64]; before that the buckets' thresholds and values, the queries' operands, and the biases [row][sub + 4]
  extern __shared__ float lds[];
  int32_t* const thr = (int32_t*)lds;
  float* const tab = lds + MAX_BUCKETS + 2;
  bf16x8* const queries = (bf16x8*)(lds + BUCKET_FLOATS);
  float* const table = lds + BUCKET_FLOATS + NQ * KS * QP * 256;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int H = p.g.H, d = EXACT ? DP : p.g.d, page = p.g.page_size;
  // (parts last: most sequences are shorter than the longest, and those without work would otherwise come at a fixed distance, which
  // leaves the working ones to a quarter of the chip: 64 sequences of power-law length up to 2048, 32 us that way)
  int idx = blockIdx.x;
  const int h = idx % H; idx /= H;
  const int qb = idx % p.qblocks; idx /= p.qblocks;
  const int b = idx % p.g.B, part = idx / p.g.B;
  const Seq s = seq_of(p, b);
  const int t0 = qb * 16 * NQ;
  if (t0 >= s.count) return;
  const int t1 = t0 + 16 * NQ < s.count ? t0 + 16 * NQ : s.count, rows = t1 - t0;
  // the block's keys: those of its last row that is there; below `all` every row attends to every key
  int end = 0, all = 0;
  {
    const int64_t last = s.place0 + t1 - 1;
    end = last < 0 || s.place0 + t0 >= s.limit ? 0 : last < s.limit ? (int)last + 1 : s.limit;
    all = last < s.limit ? keys_of(s, t0) : 0;
  }
  const int k0 = part * p.chunk;
  if (part > 0 && k0 >= end) return;
  const int k1 = end - k0 < p.chunk ? end : k0 + p.chunk;

  // (pos[j - i]: the head's entries from that of the same place on)
  const float* const pos = p.pos ? p.pos + (int64_t)(p.pos_heads > 1 ? h : 0) * (2 * (int64_t)p.max_len - 1) + p.max_len - 1 : nullptr;
  const int64_t* const ts = p.ts ? p.ts + (int64_t)b * p.max_len : nullptr;
  const Buckets buckets{thr, tab, p.ts_buckets, p.buckets_per_log2};
  if (ts) {
    for (int i = threadIdx.x; i < MAX_BUCKETS + 2; i += THREADS) thr[i] = p.thr[i];
    for (int i = threadIdx.x; i <= p.ts_buckets; i += THREADS) tab[i] = p.ts_tab[(int64_t)(p.ts_heads > 1 ? h : 0) * (p.ts_buckets + 1) + i];
  }

  const int row_bytes = d * BITS / 8, blocks = (d + 31) / 32;
  // a lane's places in a step's rows and exponents; lanes past the head's dims read its first ones (their part of Q is zeros, their rows
  // of O^T go nowhere)
  const int kg = g * (DP / 4) < d ? g : 0, vg = r * VN < d ? r : 0;
  const uint32_t k_lane = (uint32_t)((8 * (r >> 2) + (r & 3)) * row_bytes + kg * R::KB), v_lane = (uint32_t)(8 * g * row_bytes + vg * R::VB);
  const uint32_t kx_lane = (uint32_t)(kg * (DP / 4) / 32 * page + 8 * (r >> 2) + (r & 3)), vx_lane = (uint32_t)(vg * VN / 32 * page + 8 * g);
  // the head's rows and exponents in page 0, and from one page to the next
  const int64_t code_page = (int64_t)H * page * row_bytes, scale_page = (int64_t)H * blocks * page;
  const uint8_t* const k_head = (const uint8_t*)p.g.k_codes + (int64_t)h * page * row_bytes;
  const uint8_t* const v_head = (const uint8_t*)p.g.v_codes + (int64_t)h * page * row_bytes;
  const uint8_t* const kx_head = (const uint8_t*)p.g.k_scales + (int64_t)h * blocks * page;
  const uint8_t* const vx_head = (const uint8_t*)p.g.v_scales + (int64_t)h * blocks * page;

  // the page of a step's keys; steps come in order, so their page is found by counting on.  A page that is not there stands for page 0
  // with all of its keys masked, a step past the last for the last one: every step loads, whatever comes of it.
  int at_page = k0 / page, at_key = k0, slot = k0 - at_page * page, id = 0;
  bool there = false;
  auto go_to = [&](int key) {
    if (key >= k1) return;
    slot += key - at_key;
    at_key = key;
    while (slot >= page) { slot -= page; ++at_page; }
    // (a scalar load: a vector one would be waited for behind all of the step's)
    id = ((const Constant*)(uintptr_t)p.g.page_table)[(int64_t)b * p.g.table_pages + __builtin_amdgcn_readfirstlane(at_page)];
    there = id >= 0 && id < p.g.n_pages;
    id = there ? id : 0;
  };
  R x = {};
  // (the lane's part of an address stays 32 bits beside a scalar base)
  auto load_k = [&]() {
    uint32_t at = k_lane, xat = kx_lane;
    asm volatile("" : "+v"(at), "+v"(xat));
    const uint8_t* const rows = k_head + (id * code_page + slot * row_bytes);
    const uint8_t* const exps = kx_head + (id * scale_page + slot);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      x.k[t] = load_bytes<R::KB>(rows + 4 * t * row_bytes + at);
#pragma unroll
      for (int m = 0; m < R::KBLK; ++m) x.ke[t][m] = (exps + m * page + 4 * t)[xat];
    }
  };
  auto load_v = [&]() {
    uint32_t at = v_lane, xat = vx_lane;
    asm volatile("" : "+v"(at), "+v"(xat));
    const uint8_t* const rows = v_head + (id * code_page + slot * row_bytes);
    const uint2 e = *(const uint2*)(vx_head + (id * scale_page + slot) + xat);
    x.ve[0] = e.x; x.ve[1] = e.y;
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = load_bytes<R::VB>(rows + i * row_bytes + at);
  };

  const bool any = k0 < k1 && p.g.n_pages > 0;
  int next = k0 + STEP * wave;
  if (any) {
    go_to(next);
    load_k();
    load_v();
  }

  // queries, in LDS as the operands that all four waves use: lane (r, g) has row r's dims g d/4 ... of each tile
  int keys[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) keys[n] = keys_of(s, t0 + 16 * n + r);
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int64_t row = (p.offsets ? s.first * p.q_st : (int64_t)b * p.q_sb) + (int64_t)(t0 + 16 * n + r) * p.q_st + (int64_t)h * p.q_sh;
    for (int k = wave; k < KS; k += WAVES) {
      const int e = g * (DP / 4) + 8 * k;
      float y[8] = {};
      if (keys[n] > 0 && e < d) {
        if constexpr (F32) {
          const floatx4* at = (const floatx4*)((const float*)p.q + row + e);
          const floatx4 a = at[0], c = at[1];
#pragma unroll
          for (int i = 0; i < 4; ++i) { y[i] = a[i]; y[4 + i] = c[i]; }
        } else {
          unpack8(*(const uint4*)((const bf16_t*)p.q + row + e), y);
        }
      }
      bf16x8 parts[QP];
      split8<QP, true>(y, parts);
#pragma unroll
      for (int c = 0; c < QP; ++c) queries[((n * KS + k) * QP + c) * 64 + lane] = parts[c];
    }
  }

  floatx4 acc[NQ][VN];
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int j = 0; j < VN; ++j) acc[n][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  const int sub = 1 << p.sub_log2, pitch = sub + 4;
  const int place0 = (int)s.place0 + t0;              // (places of rows: lengths of at most 2^31)
  // (vmcnt(0), here and behind the biases: what the compiler does not know to have arrived when the loop begins it waits for in every
  // round of it, and with it for the loads ahead)
  __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
  for (int c0 = k0; c0 < k1; c0 += sub) {
    const int c1 = k1 - c0 < sub ? k1 : c0 + sub;
    if (ts) {
      // a pair's bias each: a thread has one key at a time and runs over the rows, or over every 2nd, 4th, ... of them
      __syncthreads();
      const int wide = p.sub_log2 < 8 ? p.sub_log2 : 8, every = THREADS >> wide;
      for (int jj = threadIdx.x & ((1 << wide) - 1); jj < c1 - c0; jj += THREADS) {
        const int j = c0 + jj;
        const int64_t tk = ts[j];
#pragma unroll 1
        for (int t = threadIdx.x >> wide; t < rows; t += every) {
          const int i = place0 + t;
          float x = 0.f;
          if (i >= j && i < s.limit) x = (pos ? pos[j - i] : 0.f) + bucket_value(buckets, ts[i < s.last_ts ? i + 1 : s.last_ts] - tk);
          table[t * pitch + jj] = x;
        }
      }
      __builtin_amdgcn_s_waitcnt(0x0f70);
      __syncthreads();
    } else if (pos) {
      // the position's alone depends on j - i: the table's entries from the last row's first key on
      __syncthreads();
      for (int e = threadIdx.x; e < c1 - c0 + rows; e += THREADS) {
        const int diff = c0 - (place0 + rows - 1) + e;
        table[e] = diff <= 0 && diff > -p.max_len ? pos[diff] : 0.f;
      }
      __builtin_amdgcn_s_waitcnt(0x0f70);
      __syncthreads();
    }
    for (int key0 = next; key0 < c1; key0 = next) {
      const int last = there ? k1 : key0;                 // (no key of a missing page is there)
      const bool whole = there && key0 + STEP <= all;
      next = key0 + STEP * WAVES;
      go_to(next);

      floatx4 st[2][NQ];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        uint32_t w[DP / 8];
#pragma unroll
        for (int m = 0; m < R::KBLK; ++m) {
          const float power = x.ke[t][m] == 255u ? __builtin_nanf("") : power_of(x.ke[t][m]);
          // (a run of two blocks: half of its bytes each)
          constexpr int HALF = R::KB / R::KBLK;
          Bytes<HALF> half;
#pragma unroll
          for (int i = 0; i < (HALF < 4 ? 1 : HALF / 4); ++i) half.w[i] = x.k[t].w[m * (HALF / 4) + i];
          pairs_of<BITS, HALF, DP / 8 / R::KBLK>(half, power, w + m * (DP / 8 / R::KBLK));
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) st[t][n] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const bf16x8 a = operand(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
#pragma unroll
          for (int n = 0; n < NQ; ++n)
            if (n == 0 || 16 * n < rows) {
#pragma unroll
              for (int c = 0; c < QP; ++c) st[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, queries[((n * KS + k) * QP + c) * 64 + lane], st[t][n], 0, 0, 0);
            }
        }
      }

      // the next step's keys are on their way while this one's weights and values are worked on, and its values after that
      load_k();

      // (copies: what the loads write stays untouched, or the compiler moves it while it is on its way and waits for it to do so)
      Bytes<R::VB> v[8];
      uint32_t ve[2] = {x.ve[0], x.ve[1]};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = x.v[i];
      // rows past the block's last key hold anything: zeros in their place
      if (key0 + STEP > last) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (key0 + 8 * g + i >= last) {
#pragma unroll
            for (uint32_t& w : v[i].w) w = 0;
            ve[i / 4] &= ~(0xffu << (8 * (i % 4)));
          }
      }
      // a value row that is not finite makes the kept weights of its key NaN (0 times it would be NaN for the others too)
      uint32_t nan_keys = 0;
      const uint32_t odd = (((ve[0] & 0x7f7f7f7fu) + 0x01010101u) & ve[0]) | (((ve[1] & 0x7f7f7f7fu) + 0x01010101u) & ve[1]);
      const bool any_nan = __any((odd & 0x80808080u) != 0);
      if (any_nan) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (((ve[i / 4] >> (8 * (i % 4))) & 0xffu) == 0xffu) {
            nan_keys |= 1u << i;
            ve[i / 4] ^= 0x80u << (8 * (i % 4));
          }
      }

      bf16x8 w8[NQ][WP];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        if (n > 0 && 16 * n >= rows) continue;
        float y[8];
        if (ts || pos) {
          const int t = 16 * n + r < rows ? 16 * n + r : rows - 1, jj = key0 - c0 + 8 * g;
          const float* const at = table + (ts ? t * pitch + jj : rows - 1 - t + jj);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(p.alpha, st[i / 4][n][i % 4], at[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = p.alpha * st[i / 4][n][i % 4];
        }
        // x sigmoid(x), a stage at a time: the transcendentals of eight keys wait for none of each other
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(-LOG2E * y[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_rcpf(1.0f + e[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= e[i];
        if (!whole || any_nan) {
          const int j0 = key0 + 8 * g;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (nan_keys >> i & 1u) y[i] = __builtin_nanf("");
            y[i] = j0 + i < keys[n] && j0 + i < last ? y[i] : 0.f;
          }
        }
        split8<WP, false>(y, w8[n]);
      }

      float power[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) power[i] = power_of((ve[i / 4] >> (8 * (i % 4))) & 0xffu);
      // dims 2 m and 2 m + 1 of the lane's run: its keys' pairs, then one operand for each
      each_pair<0, VN / 2>([&](auto m) {
        constexpr int M = decltype(m)::value;
        uint32_t pair[8], lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) pair[i] = pair_at<BITS, M>(v[i], power[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x05040100u);
          hi[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x07060302u);
        }
        const bf16x8 a0 = operand(lo[0], lo[1], lo[2], lo[3]), a1 = operand(hi[0], hi[1], hi[2], hi[3]);
#pragma unroll
        for (int n = 0; n < NQ; ++n)
          if (n == 0 || 16 * n < rows) {
#pragma unroll
            for (int c = 0; c < WP; ++c) {
              acc[n][2 * M] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, w8[n][c], acc[n][2 * M], 0, 0, 0);
              acc[n][2 * M + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, w8[n][c], acc[n][2 * M + 1], 0, 0, 0);
            }
          }
      });
      load_v();
    }
  }

  // the four waves' sums, in a fixed order: 2 and 3 onto 0 and 1, then 1 onto 0
  __syncthreads();
  auto put = [&](float* to) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int j = 0; j < VN; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) to[((n * VN + j) * 4 + i) * 64 + lane] = acc[n][j][i];
  };
  auto add = [&](const float* from) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int j = 0; j < VN; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][j][i] += from[((n * VN + j) * 4 + i) * 64 + lane];
  };
  if (wave >= 2) put(lds + (wave - 2) * ACC * 64);
  __syncthreads();
  if (wave < 2) add(lds + wave * ACC * 64);
  __syncthreads();
  if (wave == 1) put(lds);
  __syncthreads();
  if (wave != 0) return;
  add(lds);

#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int t = t0 + 16 * n + r;
    if (t >= s.count) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = (4 * g + i) * VN;        // dims e .. e + VN - 1
      if (e >= d) continue;
      if (p.partial) {
        float* to = p.partial + (((s.first + t) * H + h) * p.parts + part) * d + e;
#pragma unroll
        for (int j = 0; j < VN; j += 2) *(floatx2*)(to + j) = floatx2{acc[n][j][i], acc[n][j + 1][i]};
      } else {
        const int64_t to = (p.offsets ? s.first * p.o_st : (int64_t)b * p.o_sb) + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + e;
#pragma unroll
        for (int j = 0; j < VN; j += 2) {
          const float y0 = acc[n][j][i] * p.inv_n, y1 = acc[n][j + 1][i] * p.inv_n;
          if constexpr (F32) *(floatx2*)((float*)p.out + to + j) = floatx2{y0, y1};
          else *(uint32_t*)((bf16_t*)p.out + to + j) = pack2(y0, y1);
        }
      }
    }
  }
}

// The parts of a row, added in order: a thread has four dims of one (row, head).
template <bool F32>
__global__ __launch_bounds__(THREADS) void hstu_cached_attn_join(const Params p) {
  const int H = p.g.H, d4 = p.g.d / 4;
  const int64_t per = (int64_t)p.per_seq * H * d4;
  const int64_t groups = (per + THREADS - 1) / THREADS;
  const int b = (int)(blockIdx.x / groups);
  int64_t e = (blockIdx.x % groups) * THREADS + threadIdx.x;
  if (e >= per) return;
  const int c = (int)(e % d4); e /= d4;
  const int h = (int)(e % H), t = (int)(e / H);
  const Seq s = seq_of(p, b);
  if (t >= s.count) return;
  const int n = (keys_of(s, t) + p.chunk - 1) / p.chunk;
  const floatx4* from = (const floatx4*)(p.partial + ((s.first + t) * H + h) * p.parts * (int64_t)p.g.d) + c;
  floatx4 y = {0.f, 0.f, 0.f, 0.f};
  for (int m = 0; m < n; ++m) y += from[(int64_t)m * d4];
  const int64_t to = (p.offsets ? s.first * p.o_st : (int64_t)b * p.o_sb) + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + 4 * c;
  y *= p.inv_n;
  if constexpr (F32) *(floatx4*)((float*)p.out + to) = y;
  else *(uint2*)((bf16_t*)p.out + to) = uint2{pack2(y[0], y[1]), pack2(y[2], y[3])};
}

// The bucket law's integer thresholds up to bucket `count`: thr[b] is the smallest time difference in [1, 1e9] whose bucket
// floor(ln(fl32(dt)) / size) is b or more (INT32_MAX: none).  The last size's are kept.
void thresholds(float size, int count, int32_t* out) {
  static std::mutex lock;
  static float known = -1.f;
  static int32_t table[MAX_BUCKETS + 2];
  std::lock_guard<std::mutex> hold(lock);
  if (known != size) {
    auto bucket = [size](int32_t dt) { return floor(log((double)(float)dt) / (double)size); };
    int32_t lo = 1;
    for (int b = 0; b < MAX_BUCKETS + 2; ++b) {
      if (bucket(1000000000) < b) { table[b] = 0x7fffffff; continue; }
      int32_t x = lo, y = 1000000000;              // the answer lies in [x, y]
      while (x < y) {
        const int32_t m = x + (y - x) / 2;
        if (bucket(m) >= b) y = m; else x = m + 1;
      }
      table[b] = lo = x;
    }
    known = size;
  }
  for (int b = 0; b < MAX_BUCKETS + 2; ++b) out[b] = b <= count ? table[b] : 0x7fffffff;
}

struct Split { int nq, qblocks, parts, chunk; };

// How a call is cut up, by its sizes alone (the lengths are on the device).
Split split_of(const HstuCachedAttnArgs& a) {
  Split s;
  const bool f32 = a.dtype == HSTU_SERVE_FP32;
  const int most = a.pages.d > 128 ? (f32 ? 1 : 2) : f32 ? 2 : 4;
  // blocks of 16, 32 or 64 rows, by how many a sequence has: a step of keys is converted once for a block's rows, and the more they are the fewer
  // waves a SIMD holds.  128 sequences of 1024 keys, 8 heads, 4 bits, bf16, both tables, on blocks of 16 / 32 / 64: head dims of 64, 24 rows
  // 89 / 73 / 107 us, 64 rows 168 / 154 / 221; of 128, 24 rows 103 / 108 / 220, 64 rows 191 / 198 / 450; 4 heads of 256, 24 rows 94 / 143, 64 rows
  // 179 / 270.  With positions alone: 64, 24 rows 37 / 32 / 47; 128, 24 rows 49 / 51 / 106, 64 rows 91 / 84 / 144.  So two blocks of 32 beat one of 64
  // wherever it is taken, and 16 rows beat 32 at head dims of 256 and, with times, mostly at 128.
  s.nq = a.rows_per_seq > 32 ? 4 : a.rows_per_seq > 16 ? 2 : 1;
  s.nq = std::min(s.nq, most);
  s.qblocks = (a.rows_per_seq + 16 * s.nq - 1) / (16 * s.nq);
  const int64_t cap = std::min<int64_t>(a.max_len, (int64_t)a.pages.table_pages * a.pages.page_size);
  const int64_t base = (int64_t)a.pages.B * a.pages.H * s.qblocks;
  // 2048 workgroups, of 256 keys at least and of 1024 where there are many without splitting: a part costs its start and the join's launch
  // (512 sequences of 512 keys: one part 12.9 us, two 15.8), a long one that the others wait for it.  64 sequences x 8 heads, up to 2048 keys of 128 in 4
  // bits: 4 parts 16.4 us at power-law lengths and 36.4 at full ones, 2 parts 18.4 and 33.4, one 20.4 and 33.7, 8 parts 18.2 and 43.
  const int64_t least = std::max<int64_t>(256, std::min<int64_t>(base, 1024));
  const int64_t parts = std::max<int64_t>(1, std::min((2048 + base - 1) / base, (cap + least - 1) / least));
  const int64_t chunk = std::max<int64_t>(128, ((cap + parts - 1) / parts + 127) / 128 * 128);
  s.chunk = (int)std::min<int64_t>(chunk, 1 << 30);
  s.parts = (int)std::max<int64_t>(1, (cap + s.chunk - 1) / s.chunk);
  return s;
}

int check(const HstuCachedAttnArgs* a) {
  if (!a) return serve_fail(HSTU_SERVE_ERR_NULL, "args is null");
  if (a->struct_size != sizeof(HstuCachedAttnArgs) || a->version != HSTU_SERVE_ABI_VERSION)
    return serve_fail(HSTU_SERVE_ERR_VERSION, "struct_size %u version %u, expected %zu and %d", a->struct_size, a->version, sizeof(HstuCachedAttnArgs), HSTU_SERVE_ABI_VERSION);
  if (const int rc = serve_check_pages(a->pages)) return rc;
  if (a->dtype != HSTU_SERVE_BF16 && a->dtype != HSTU_SERVE_FP32) return serve_fail(HSTU_SERVE_ERR_SHAPE, "dtype %d", a->dtype);
  if (a->rows_per_seq < 0 || a->total_rows < 0 || a->max_len < 1) return serve_fail(HSTU_SERVE_ERR_SHAPE, "rows_per_seq=%d total_rows=%lld max_len=%d", a->rows_per_seq, (long long)a->total_rows, a->max_len);
  if (a->max_len > 1 << 30 || a->rows_per_seq > 1 << 30) return serve_fail(HSTU_SERVE_ERR_SHAPE, "rows_per_seq=%d max_len=%d: at most 2^30", a->rows_per_seq, a->max_len);
  if (a->pos_tab && a->pos_heads != 1 && a->pos_heads != a->pages.H) return serve_fail(HSTU_SERVE_ERR_SHAPE, "pos_heads=%d: 1 or %d", a->pos_heads, a->pages.H);
  if (a->timestamps) {
    if (!a->ts_tab) return serve_fail(HSTU_SERVE_ERR_NULL, "ts_tab is null");
    if (a->ts_heads != 1 && a->ts_heads != a->pages.H) return serve_fail(HSTU_SERVE_ERR_SHAPE, "ts_heads=%d: 1 or %d", a->ts_heads, a->pages.H);
    if (a->ts_buckets < 0 || a->ts_buckets > MAX_BUCKETS) return serve_fail(HSTU_SERVE_ERR_SHAPE, "ts_buckets=%d: at most %d", a->ts_buckets, MAX_BUCKETS);
    if (!(a->ts_bucket_size > 0.f)) return serve_fail(HSTU_SERVE_ERR_SHAPE, "ts_bucket_size must be positive");
  }
  return HSTU_SERVE_OK;
}

bool nothing(const HstuCachedAttnArgs& a) { return a.pages.B == 0 || a.rows_per_seq == 0 || (a.offsets && a.total_rows == 0); }

size_t workspace_of(const HstuCachedAttnArgs& a, const Split& s) {
  if (s.parts == 1) return 0;
  const int64_t rows = a.offsets ? a.total_rows : (int64_t)a.pages.B * a.rows_per_seq;
  return (size_t)rows * a.pages.H * s.parts * a.pages.d * sizeof(float);
}

template <int DP, bool EXACT, int BITS, bool F32, int NQ>
void launch(const Params& p, uint32_t grid, hipStream_t st) {
  constexpr int ACC = DP / 16 * 4 * NQ;
  const int rows = std::min(p.per_seq, 16 * NQ);
  const size_t biases = p.ts ? (size_t)rows * ((1 << p.sub_log2) + 4) : p.pos ? (size_t)std::min(1 << p.sub_log2, p.chunk) + rows + 8 : 0;
  const size_t lds = std::max<size_t>((size_t)2 * ACC * 64, BUCKET_FLOATS + NQ * (DP / 32) * (F32 ? 3 : 1) * 256 + biases) * sizeof(float);
  hstu_cached_attn_kernel<DP, EXACT, BITS, F32, NQ><<<grid, THREADS, lds, st>>>(p);
}

template <int DP, bool EXACT, int BITS>
void launch_nq(const Params& p, bool f32, int nq, uint32_t grid, hipStream_t st) {
  if (f32) {
    if constexpr (DP <= 128) { if (nq == 2) return launch<DP, EXACT, BITS, true, 2>(p, grid, st); }
    return launch<DP, EXACT, BITS, true, 1>(p, grid, st);
  }
  if constexpr (DP <= 128) { if (nq == 4) return launch<DP, EXACT, BITS, false, 4>(p, grid, st); }
  if (nq == 2) return launch<DP, EXACT, BITS, false, 2>(p, grid, st);
  launch<DP, EXACT, BITS, false, 1>(p, grid, st);
}

// Head dims that are no power of two (and those below 32) run as the next one with the lanes' addresses cut off.
template <int DP, int BITS>
void launch_exact(const Params& p, bool f32, int nq, uint32_t grid, hipStream_t st) {
  if (p.g.d == DP) launch_nq<DP, true, BITS>(p, f32, nq, grid, st);
  else launch_nq<DP, false, BITS>(p, f32, nq, grid, st);
}

template <int BITS>
void launch_width(const Params& p, bool f32, int nq, uint32_t grid, hipStream_t st) {
  if (p.g.d <= 32) launch_exact<32, BITS>(p, f32, nq, grid, st);
  else if (p.g.d <= 64) launch_exact<64, BITS>(p, f32, nq, grid, st);
  else if (p.g.d <= 128) launch_exact<128, BITS>(p, f32, nq, grid, st);
  else launch_exact<256, BITS>(p, f32, nq, grid, st);
}

}  // namespace

extern "C" {

size_t hstu_cached_attn_workspace_bytes(const HstuCachedAttnArgs* a) {
  serve_clear_error();
  if (check(a) || nothing(*a)) return 0;
  return workspace_of(*a, split_of(*a));
}

int hstu_cached_attn(const HstuCachedAttnArgs* a, void* stream) {
  serve_clear_error();
  if (const int rc = check(a)) return rc;
  if (nothing(*a)) return HSTU_SERVE_OK;
  if (!a->lengths || !a->q || !a->out) return serve_fail(HSTU_SERVE_ERR_NULL, "lengths, q or out is null");
  const int64_t unit = a->dtype == HSTU_SERVE_FP32 ? 4 : 8;
  for (const void* t : {a->q, (const void*)a->out})
    if (!serve_aligned16(t)) return serve_fail(HSTU_SERVE_ERR_SHAPE, "q and out start on 16-byte boundaries");
  for (const int64_t st : {a->q_stride_t, a->q_stride_h, a->o_stride_t, a->o_stride_h, a->offsets ? (int64_t)0 : a->q_stride_b, a->offsets ? (int64_t)0 : a->o_stride_b})
    if (st % unit) return serve_fail(HSTU_SERVE_ERR_SHAPE, "a stride of %lld elements: rows start on 16-byte boundaries", (long long)st);
  const Split s = split_of(*a);
  const size_t need = workspace_of(*a, s);
  if (need && (!a->workspace || a->workspace_bytes < need || !serve_aligned16(a->workspace)))
    return serve_fail(HSTU_SERVE_ERR_WORKSPACE, "workspace of %zu bytes on a 16-byte boundary needed, got %zu", need, a->workspace_bytes);
  const int64_t grid = (int64_t)a->pages.B * a->pages.H * s.qblocks, most = SERVE_THREADS / THREADS;
  const int64_t per = (int64_t)a->rows_per_seq * a->pages.H * (a->pages.d / 4), join = (per + THREADS - 1) / THREADS * a->pages.B;
  if (grid > most / s.parts || join > most) return serve_fail(HSTU_SERVE_ERR_SHAPE, "too many workgroups for one call");
  Params p;
  p.g = a->pages;
  p.lengths = a->lengths; p.offsets = a->offsets;
  p.q = a->q; p.out = a->out;
  p.total = a->total_rows;
  p.q_sb = a->q_stride_b; p.q_st = a->q_stride_t; p.q_sh = a->q_stride_h;
  p.o_sb = a->o_stride_b; p.o_st = a->o_stride_t; p.o_sh = a->o_stride_h;
  p.pos = a->pos_tab; p.ts = a->timestamps; p.ts_tab = a->ts_tab;
  p.partial = s.parts > 1 ? (float*)a->workspace : nullptr;
  p.per_seq = a->rows_per_seq; p.max_len = a->max_len; p.pos_heads = a->pos_heads; p.ts_heads = a->ts_heads; p.ts_buckets = a->ts_buckets;
  p.chunk = s.chunk; p.parts = s.parts; p.qblocks = s.qblocks;
  // biases of 8192 pairs at a time, and of 2048 keys at most; of positions alone, of 8192 keys
  p.sub_log2 = a->timestamps ? 11 : 13;
  while (a->timestamps && p.sub_log2 > 7 && ((int64_t)std::min(a->rows_per_seq, 16 * s.nq) << p.sub_log2) > 8192) --p.sub_log2;
  p.alpha = a->alpha; p.inv_n = a->inv_n; p.buckets_per_log2 = 0.f;
  if (a->timestamps) {
    thresholds(a->ts_bucket_size, a->ts_buckets, p.thr);
    p.buckets_per_log2 = (float)(0.69314718055994530942 / (double)a->ts_bucket_size);
  }
  hipStream_t st = (hipStream_t)stream;
  const bool f32 = a->dtype == HSTU_SERVE_FP32;
  if (a->pages.bits == 4) launch_width<4>(p, f32, s.nq, (uint32_t)(grid * s.parts), st);
  else launch_width<8>(p, f32, s.nq, (uint32_t)(grid * s.parts), st);
  if (const int rc = serve_launched("hstu_cached_attn")) return rc;
  if (s.parts > 1) {
    if (f32) hstu_cached_attn_join<true><<<(uint32_t)join, THREADS, 0, st>>>(p);
    else hstu_cached_attn_join<false><<<(uint32_t)join, THREADS, 0, st>>>(p);
    return serve_launched("hstu_cached_attn_join");
  }
  return HSTU_SERVE_OK;
}

}
