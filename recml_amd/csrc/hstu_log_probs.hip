// Log probabilities of given tokens from rows of logits, with the rows' entropy and their largest entries, and the
// gradient of all of these, for gfx950 (MI355X): see include/hstu_serve.h.
//
//   lse = m + ln s,  s = sum_j exp(x_j - m),  m = max_j x_j        lp_c = (x_c - m) - ln s
//   entropy = ln s - t / s,  t = sum_j (x_j - m) exp(x_j - m)
//   d/dx_j = -p_j (G + g_e (x_j - lse + entropy)) + the gradients given for j,  G = their sum over the row
//
// Each pass reads the logits once.  A workgroup takes up to 8 vectors of 16 bytes per thread and keeps them in registers: the
// maximum is known before the first exponential, so nothing is rescaled, and the largest entries are looked for without reading
// again.  Rows that are longer are split; a second kernel joins the parts in their order.  Memory bounds all of it where there is much:
// 8192 rows of 100000 in bf16, with the entropy, forward in 305 us (5.4 TB/s) and the join in 7, backward in 600 (5.5 TB/s, as much
// written as read; both streams go past the caches, through them the three took 920 together and 850 so).  Few rows are chains of
// latencies: one of a million with its 10 largest 7.7 us and 5.5 for the join.
//
// The largest entries of a part: the k-th largest of the threads' maxima bounds the k-th largest entry from below, few entries
// reach it, and each of those finds its rank by counting who comes before it (by value, then by index).  The bound comes from
// ballots on 16 bits of the ordered value.  Where more reach it than the lists hold (ties, mostly), the k-th entry is found exactly,
// bit by bit.  4096 rows of 20011 in fp32 (328 MB) take 78 us with the 5 largest, 61 without.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "hstu_serve_common.h"

namespace {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int VECS = 8;              // vectors of 16 bytes that a thread holds
constexpr int MAX_TOP = 256;

struct Params {
  const void* logits;
  int64_t stride;
  const int64_t* tokens;             // [rows][count]
  float* log_probs;                  // [rows][count]
  float* entropy;                    // [rows] or null
  float* stats;                      // [rows][3]: m, ln s, entropy
  float* top_log_probs;              // [rows][top]
  int64_t* top_tokens;               // [rows][top]
  // one part of a row: m, s, t, and its largest entries
  float* part_stats;                 // [rows][parts][3]
  float* part_value;                 // [rows][parts][top]
  int32_t* part_index;
  // the backward
  const float* g_tokens;
  const float* g_entropy;
  const float* g_top;
  void* d_logits;
  int64_t d_stride;
  int64_t rows;
  int32_t vocab, count, top, parts, vecs;
  int32_t sums_t;                    // the entropy is wanted
};

// ordered bits: larger floats have larger ones, any NaN the largest; -0 and 0 are one value
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return x != x ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
}

// an entry's place in the order: by value, then by the lower index
__device__ __forceinline__ uint64_t place_of(float x, int index) { return (uint64_t)ordered(x) << 32 | (uint32_t)(0x7fffffff - index); }

template <bool F32>
struct Vec {
  static constexpr int N = F32 ? 4 : 8;
  uint4 raw;
  // Keeps the entries packed: without it the compiler holds them unpacked from one pass over the registers to the next (256
  // registers, one wave a SIMD).
  __device__ __forceinline__ void hold() { asm volatile("" : "+v"(raw.x), "+v"(raw.y), "+v"(raw.z), "+v"(raw.w)); }
  __device__ __forceinline__ float at(int i) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (F32) return __builtin_bit_cast(float, w[i]);
    else return __builtin_bit_cast(float, i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};

// Where a row's vectors lie: the row may start anywhere, its vectors are the memory's 16-byte pieces.  Vector v holds entries
// v N - shift ..., those outside [0, vocab) belong to somebody else and are neither read nor written.
template <bool F32>
struct Row {
  const char* base;
  int shift, vectors, vocab;
  __device__ __forceinline__ Row(const void* logits, int64_t stride, int64_t row, int n) {
    constexpr int N = Vec<F32>::N, SIZE = F32 ? 4 : 2;
    const char* at = (const char*)logits + row * stride * SIZE;
    shift = (int)((uintptr_t)at & 15u) / SIZE;
    base = at - shift * SIZE;
    vocab = n;
    vectors = (int)(((int64_t)n + shift + N - 1) / N);
  }
  __device__ __forceinline__ int first(int v) const { return v * Vec<F32>::N - shift; }
  __device__ __forceinline__ bool whole(int v) const { return first(v) >= 0 && (int64_t)first(v) + Vec<F32>::N <= vocab; }
  __device__ __forceinline__ Vec<F32> load(int v) const {
    constexpr int N = Vec<F32>::N;
    Vec<F32> r;
    if (whole(v)) {
      r.raw = __builtin_bit_cast(uint4, __builtin_nontemporal_load((const uint4v*)(base + (int64_t)v * 16)));
      return r;
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = F32 ? 0xff800000u : 0xff80ff80u;     // -inf
    const int e = first(v);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (v >= vectors || e + i < 0 || e + i >= vocab) continue;
      if constexpr (F32) w[i] = *(const uint32_t*)(base + (int64_t)v * 16 + 4 * i);
      else {
        const uint32_t half = *(const uint16_t*)(base + (int64_t)v * 16 + 2 * i);
        w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | half << 16 : (w[i / 2] & 0xffff0000u) | half;
      }
    }
    r.raw = uint4{w[0], w[1], w[2], w[3]};
    return r;
  }
};

template <int NT, typename F>
__device__ __forceinline__ float block_reduce(float x, float* lds, F op) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x = op(x, __shfl_xor(x, m, 64));
  if constexpr (NT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) x = op(x, lds[w]);
  }
  return x;
}

__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }

// What select_top shares; CAP: entries that reach the bound at most, on the short way.
template <int CAP_>
struct Chosen {
  static constexpr int CAP = CAP_;
  uint64_t place[CAP];
  float value[CAP];
  uint32_t bound[4][2];
  int n, vectors;
};

// The j-th and the k-th largest of a wave's values by the upper 16 of their ordered bits, lower bits zero (0: there are fewer).
__device__ __forceinline__ void kth_of_wave(uint32_t key, int j, int k, uint32_t* jth, uint32_t* kth) {
  uint32_t a = 0, b = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t na = a | 1u << bit, nb = b | 1u << bit;
    a = __popcll(__ballot(key >= na)) >= j ? na : a;
    b = __popcll(__ballot(key >= nb)) >= k ? nb : b;
  }
  *jth = a;
  *kth = b;
}

// The k entries themselves, where too many reach the bound: the k-th largest value bit by bit, then, among its equals, the index up
// to which they belong to the k.  Each bit is a pass over the entries: bf16's values have their upper 16 only, indices those of `vocab`.
template <bool F32, int NT, typename C, typename Each>
__device__ __forceinline__ void exactly(int k, int vocab, C& c, Each each) {
  constexpr int W = NT / 64;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  auto count = [&](auto counts) {
    int mine = 0;
    each([&](float x, int index) { mine += counts(ordered(x), index) ? 1 : 0; });
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) mine += __shfl_xor(mine, m, 64);
    if constexpr (W > 1) {
      __syncthreads();
      if (lane == 0) c.bound[wave][0] = (uint32_t)mine;
      __syncthreads();
      mine = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) mine += (int)c.bound[w][0];
    }
    return mine;
  };
  uint32_t value = 0;
#pragma unroll 1
  for (int bit = 31; bit >= (F32 ? 0 : 16); --bit) {
    const uint32_t next = value | 1u << bit;
    if (count([&](uint32_t o, int) { return o >= next; }) >= k) value = next;
  }
  if (!F32 && (value < 0x80000000u || value == 0xffff0000u)) value |= 0xffffu;      // (negative ones' lower bits, and a NaN's)
  const int ties = k - count([&](uint32_t o, int) { return o > value; });
  int below = 0;                           // the largest index with fewer than `ties` equals below it
#pragma unroll 1
  for (int bit = 31 - __builtin_clz(vocab); bit >= 0; --bit) {
    const int next = below | 1 << bit;
    if (count([&](uint32_t o, int index) { return o == value && index < next; }) < ties) below = next;
  }
  __syncthreads();
  if (threadIdx.x == 0) c.n = 0;
  __syncthreads();
  each([&](float x, int index) {
    const uint32_t o = ordered(x);
    if (o > value || (o == value && index <= below)) {
      const int at = atomicAdd(&c.n, 1);
      c.place[at] = place_of(x, index);    // (k of them)
      c.value[at] = x;
    }
  });
  __syncthreads();
}

// The k largest of the workgroup's entries, the r-th of them given to out(r, value, index).  `most`: the ordered bits of a
// thread's largest entry (0: it has none; the least of an entry is that of -inf); collect(bound, reaches, push), called by all threads,
// calls push(x, index) for the entries that reach the bound, each(f) f(x, index) for all of a thread's; there are at least k.
template <bool F32, int NT, typename C, typename Collect, typename Each, typename Out>
__device__ __forceinline__ void select_top(int k, int vocab, C& c, uint32_t most, Collect collect, Each each, Out out) {
  constexpr int W = NT / 64;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  // every wave has its share of the k, or one wave has all of them: either way k entries reach the bound.  (The shares bound well
  // where all waves are full, the wave's k where one of them holds little.)
  uint32_t share, all;
  kth_of_wave(most, (k + W - 1) / W, k, &share, &all);
  uint32_t bound = share;
  if constexpr (W > 1) {
    if (lane == 0) { c.bound[wave][0] = share; c.bound[wave][1] = all; }
    __syncthreads();
    uint32_t best = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      bound = c.bound[w][0] < bound ? c.bound[w][0] : bound;
      best = c.bound[w][1] > best ? c.bound[w][1] : best;
    }
    bound = best > bound ? best : bound;
  }
  if (threadIdx.x == 0) c.n = c.vectors = 0;
  __syncthreads();
  collect(bound, most != 0 && most >= bound, [&](float x, int index) {
    const int at = atomicAdd(&c.n, 1);
    if (at < C::CAP) { c.place[at] = place_of(x, index); c.value[at] = x; }
  });
  __syncthreads();
  int n = c.n;
  if (n > C::CAP) {
    exactly<F32, NT>(k, vocab, c, each);
    n = k;
  }
  // who comes before an entry is its rank
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t mine = c.place[i];
    int before = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) before += c.place[j] > mine;
    if (before < k) out(before, c.value[i], 0x7fffffff - (int)(uint32_t)mine);
  }
  __syncthreads();
}

// m + ln s and the entropy of a row from its sums; m = -inf stands for a row without any finite entry.
__device__ __forceinline__ float entropy_of(float log_s, float s, float t) { return log_s - t / s; }

template <bool F32>
__device__ __forceinline__ float logit_at(const Params& p, int64_t row, int64_t index) {
  const int64_t at = row * p.stride + index;
  if constexpr (F32) return ((const float*)p.logits)[at];
  else return (float)((const bf16_t*)p.logits)[at];
}

// A thread's first token of a row and its logit, asked for ahead of the sums.
struct First { int64_t token; float logit; };

template <bool F32>
__device__ __forceinline__ First first_of(const Params& p, int64_t row) {
  First f = {-1, 0.f};
  if ((int)threadIdx.x < p.count) f.token = p.tokens[row * p.count + threadIdx.x];
  if (f.token >= 0 && f.token < p.vocab) f.logit = logit_at<F32>(p, row, f.token);
  return f;
}

// What is asked of a row once its sums are known.
template <bool F32, int NT>
__device__ __forceinline__ void finish(const Params& p, int64_t row, float m, float s, float t, const First& first) {
  // (NaN where t was not summed: a backward that asks for the entropy's part all the same shows it)
  const float log_s = __logf(s), entropy = p.sums_t ? entropy_of(log_s, s, t) : __builtin_nanf("");
  if (threadIdx.x == 0) {
    if (p.stats) { p.stats[row * 3] = m; p.stats[row * 3 + 1] = log_s; p.stats[row * 3 + 2] = entropy; }
    if (p.entropy) p.entropy[row] = entropy;
  }
  for (int c = threadIdx.x; c < p.count; c += NT) {
    const bool early = c < NT;
    const int64_t token = early ? first.token : p.tokens[row * p.count + c];
    float y = 0.f;                                             // (nothing asked)
    if (token >= p.vocab) y = __builtin_nanf("");
    else if (token >= 0) y = ((early ? first.logit : logit_at<F32>(p, row, token)) - m) - log_s;
    p.log_probs[row * p.count + c] = y;
  }
}

template <bool F32, int NT, bool TOP>
__global__ __launch_bounds__(NT) void hstu_log_probs_part(const Params p) {
  constexpr int N = Vec<F32>::N;
  __shared__ float sums[4];
  const int64_t row = blockIdx.x / p.parts;
  const int part = blockIdx.x % p.parts;
  const Row<F32> r(p.logits, p.stride, row, p.vocab);
  const int v0 = part * p.vecs * NT + threadIdx.x;
  Vec<F32> x[VECS];
#pragma unroll
  for (int c = 0; c < VECS; ++c)
    if (c < p.vecs) x[c] = r.load(v0 + c * NT);
  float m = -__builtin_inff();
#pragma unroll
  for (int c = 0; c < VECS; ++c)
    if (c < p.vecs) {
#pragma unroll
      for (int i = 0; i < N; ++i) m = fmaxf(m, x[c].at(i));
      x[c].hold();
    }
  const float mine = m;
  m = block_reduce<NT>(m, sums, larger);
  const float zero = m == -__builtin_inff() ? 0.f : m;         // (a part without any entry above -inf sums to nothing)
  float s = 0.f, t = 0.f;
  if (p.sums_t) {
#pragma unroll
    for (int c = 0; c < VECS; ++c)
      if (c < p.vecs) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float d = x[c].at(i) - zero, e = __builtin_amdgcn_exp2f(d * LOG2E);
          s += e;
          t = __builtin_fmaf(fmaxf(d, -1e4f), e, t);           // (e is 0 long before: -inf times its 0 is nothing; a NaN is in s)
        }
        x[c].hold();
      }
    t = block_reduce<NT>(t, sums, add);
  } else {
#pragma unroll
    for (int c = 0; c < VECS; ++c)
      if (c < p.vecs) {
#pragma unroll
        for (int i = 0; i < N; ++i) s += __builtin_amdgcn_exp2f((x[c].at(i) - zero) * LOG2E);
        x[c].hold();
      }
  }
  const bool odd = s != s;             // (the thread holds a NaN, or +inf)
  s = block_reduce<NT>(s, sums, add);
  if (p.parts == 1) {
    finish<F32, NT>(p, row, m, s, t, first_of<F32>(p, row));     // (earlier, it costs a wave a SIMD)
  } else if (threadIdx.x == 0) {
    float* to = p.part_stats + (row * p.parts + part) * 3;
    to[0] = m; to[1] = s; to[2] = t;
  }
  if constexpr (!TOP) return;
  __shared__ Chosen<NT == 64 ? 256 : 1024> chosen;
  constexpr int HELD = NT == 64 ? 192 : 512;                   // vectors with entries that reach the bound
  __shared__ uint4 held[HELD];
  __shared__ int32_t held_at[HELD];
  // a part shorter than `top` gives what it has
  const int64_t e0 = (int64_t)part * p.vecs * NT * N - r.shift, e1 = e0 + (int64_t)p.vecs * NT * N;
  const int64_t here = (e1 < p.vocab ? e1 : p.vocab) - (e0 > 0 ? e0 : 0);
  const int k = here < p.top ? (here > 0 ? (int)here : 0) : p.top;
  const float log_s = __logf(s);
  // (read again: from the registers the long way would hold their ordered bits too, and cost the short one a third of its waves)
  auto each = [&](auto f) {
#pragma unroll 1
    for (int c = 0; c < p.vecs; ++c) {
      const int v = v0 + c * NT, e = r.first(v);
      const Vec<F32> y = r.load(v);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (v < r.vectors && e + i >= 0 && e + i < p.vocab) f(y.at(i), e + i);
    }
  };
  uint32_t most = v0 < r.vectors ? ordered(mine) : 0;
  if (odd) each([&](float y, int) { const uint32_t o = ordered(y); most = o > most ? o : most; });
  auto collect = [&](uint32_t bound, bool reaches, auto push) {
    // vectors with an entry that is not below the bound's float (where that is a NaN, all of them), then their entries: the code that
    // an entry takes is there once, not 64 times (which is fetched on every launch, a third of a small call's time)
    const float least = __builtin_bit_cast(float, bound & 0x80000000u ? bound & 0x7fffffffu : ~bound);
    if (reaches) {
#pragma unroll
      for (int c = 0; c < VECS; ++c)
        if (c < p.vecs) {
          bool any = false;
          x[c].hold();
#pragma unroll
          for (int i = 0; i < N; ++i) any |= !(x[c].at(i) < least);
          if (any) {
            const int at = atomicAdd(&chosen.vectors, 1);
            if (at < HELD) { held[at] = x[c].raw; held_at[at] = r.first(v0 + c * NT); }
          }
        }
    }
    __syncthreads();
    const int n = chosen.vectors;
    if (n > HELD) {                                            // (all the same to the bound: the long way)
      if (threadIdx.x == 0) chosen.n = 1 << 30;
      return;
    }
    for (int i = threadIdx.x; i < n * N; i += NT) {
      const int e = held_at[i / N] + i % N;
      const uint32_t w = ((const uint32_t*)held)[F32 ? i : i / 2];
      const float y = __builtin_bit_cast(float, F32 ? w : i % 2 ? w & 0xffff0000u : w << 16);
      if (e >= 0 && e < p.vocab && ordered(y) >= bound) push(y, e);
    }
  };
  const int64_t to = (row * p.parts + part) * p.top;
  if (p.parts > 1)
    for (int i = k + threadIdx.x; i < p.top; i += NT) p.part_index[to + i] = -1;
  if (k > 0)
    select_top<F32, NT>(k, p.vocab, chosen, most, collect, each, [&](int rank, float value, int index) {
      if (p.parts == 1) {
        p.top_log_probs[to + rank] = (value - m) - log_s;
        p.top_tokens[to + rank] = index;
      } else {
        p.part_value[to + rank] = value;
        p.part_index[to + rank] = index;
      }
    });
}

// One row's parts: their sums in order, and the largest of their largest.
template <bool F32, int NT>
__global__ __launch_bounds__(NT) void hstu_log_probs_join(const Params p) {
  constexpr int E = NT == 64 ? 4 : 8, TOP = NT == 64 ? 64 : MAX_TOP;
  __shared__ Chosen<NT * E> chosen;
  __shared__ float sums[4];
  __shared__ float best_value[TOP];
  __shared__ int32_t best_index[TOP];
  const int64_t row = blockIdx.x;
  const float* from = p.part_stats + row * p.parts * 3;
  // (a row is a chain of latencies: what does not depend on the sums is asked for ahead of them)
  const int64_t base = row * p.parts * p.top, total = (int64_t)p.parts * p.top;
  float x[E];
  int index[E];
  auto fetch = [&](int64_t done, int have, int take) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = e * NT + threadIdx.x - have;
      if (i < 0) continue;
      index[e] = -1;
      x[e] = 0.f;
      if (i < take) { index[e] = p.part_index[base + done + i]; x[e] = p.part_value[base + done + i]; }
    }
  };
  int take = total < NT * E ? (int)total : NT * E;
  fetch(0, 0, take);
  const First first = first_of<F32>(p, row);
  float m = -__builtin_inff();
  for (int i = threadIdx.x; i < p.parts; i += NT) m = fmaxf(m, from[3 * i]);
  m = block_reduce<NT>(m, sums, larger);
  const float zero = m == -__builtin_inff() ? 0.f : m;
  float s = 0.f, t = 0.f;
  for (int i = threadIdx.x; i < p.parts; i += NT) {
    // a part's sums are about its own maximum: sum (x - m) e = scale (t + (its m - m) s)
    const float d = from[3 * i] - zero, scale = __builtin_amdgcn_exp2f(d * LOG2E), ps = from[3 * i + 1];
    s += scale * ps;
    t += scale > 0.f ? scale * (from[3 * i + 2] + d * ps) : ps == ps ? 0.f : ps;
  }
  s = block_reduce<NT>(s, sums, add);
  t = block_reduce<NT>(t, sums, add);
  finish<F32, NT>(p, row, m, s, t, first);
  if (p.top == 0) return;
  const float log_s = __logf(s);
  int have = 0;                        // the best of the entries so far, in LDS
  for (int64_t done = 0; done < total;) {
    if (done > 0) {
      take = total - done < NT * E - have ? (int)(total - done) : NT * E - have;
      fetch(done, have, take);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = e * NT + threadIdx.x;
        if (i < have) { x[e] = best_value[i]; index[e] = best_index[i]; }
      }
      __syncthreads();
    }
    float there = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) there += index[e] >= 0 ? 1.f : 0.f;
    const int n = (int)block_reduce<NT>(there, sums, add);
    const int k = n < p.top ? n : p.top;
    done += take;
    const bool end = done >= total;
    auto each = [&](auto f) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (index[e] >= 0) f(x[e], index[e]);
    };
    uint32_t most = 0;
    each([&](float y, int) { const uint32_t o = ordered(y); most = o > most ? o : most; });
    auto collect = [&](uint32_t bound, bool reaches, auto push) {
      if (reaches) each([&](float y, int i) { if (ordered(y) >= bound) push(y, i); });
    };
    if (k > 0)
      select_top<F32, NT>(k, p.vocab, chosen, most, collect, each, [&](int rank, float value, int at) {
        if (end) {
          p.top_log_probs[row * p.top + rank] = (value - m) - log_s;
          p.top_tokens[row * p.top + rank] = at;
        } else {
          best_value[rank] = value;
          best_index[rank] = at;
        }
      });
    have = k;
    __syncthreads();
  }
}

template <bool F32, int NT>
__global__ __launch_bounds__(NT) void hstu_log_probs_backward(const Params p) {
  constexpr int N = Vec<F32>::N, SIZE = F32 ? 4 : 2;
  __shared__ uint32_t hit[NT * VECS * N / 32], several[NT * VECS * N / 32];
  constexpr int LIST = 4 * NT;
  // the places of the first outputs' entries in the part, and their gradients
  __shared__ __attribute__((aligned(16))) int list[LIST];
  __shared__ __attribute__((aligned(16))) float gradient[LIST];
  __shared__ uint16_t queue[LIST];     // those whose entries are others' too
  __shared__ int queued, repeated;
  __shared__ float sums[4];
  const int64_t row = blockIdx.x / p.parts;
  const int part = blockIdx.x % p.parts;
  const Row<F32> r(p.logits, p.stride, row, p.vocab);
  const int v0 = part * p.vecs * NT;
  Vec<F32> x[VECS];
#pragma unroll
  for (int c = 0; c < VECS; ++c)
    if (c < p.vecs) x[c] = r.load(v0 + c * NT + threadIdx.x);
  // the gradients' sum, and which of the part's entries have one of their own, or several
  const int64_t e0 = (int64_t)v0 * N - r.shift;
  const int entries = NT * p.vecs * N, asked = (p.g_tokens ? p.count : 0) + (p.g_top ? p.top : 0), given = p.g_tokens ? p.count : 0;
  for (int i = threadIdx.x; i < entries / 32; i += NT) hit[i] = several[i] = 0;
  if (threadIdx.x == 0) queued = repeated = 0;
  __syncthreads();
  // (the c-th of the outputs: the tokens', then the largest entries')
  auto index_of = [&](int c) { return c < given ? p.tokens[row * p.count + c] : p.top_tokens[row * p.top + c - given]; };
  auto gradient_of = [&](int c) { return c < given ? p.g_tokens[row * p.count + c] : p.g_top[row * p.top + c - given]; };
  float total = 0.f;
  // (which of the part's entries an index is; -1: none)
  auto place_in = [&](int64_t index) { return index >= 0 && index < p.vocab && index >= e0 && index - e0 < entries ? (int)(index - e0) : -1; };
  auto mark = [&](int c) {
    const int64_t index = index_of(c);
    const int at = place_in(index);
    const float g = index < 0 ? 0.f : index < p.vocab ? gradient_of(c) : __builtin_nanf("");
    total += g;
    if (at >= 0) {
      const uint32_t bit = 1u << (at % 32);
      if (atomicOr(&hit[at / 32], bit) & bit) {
        atomicOr(&several[at / 32], bit);
        repeated = 1;
      }
    }
    if (c < LIST) { list[c] = at; gradient[c] = g; }
    return at;
  };
  // (the thread's first one outside the loop: its logit is on its way from here on)
  int mine = -1;
  float early = 0.f;
  if (threadIdx.x < asked) mine = mark(threadIdx.x);
  if (mine >= 0) early = logit_at<F32>(p, row, e0 + mine);
  for (int c = threadIdx.x + NT; c < asked; c += NT) mark(c);
  for (int c = asked + threadIdx.x; c < LIST && c < (asked + 7) / 8 * 8; c += NT) { list[c] = -1; gradient[c] = 0.f; }
  total = block_reduce<NT>(total, sums, add);
  __syncthreads();
  const float m = p.stats[row * 3], log_s = p.stats[row * 3 + 1], entropy = p.stats[row * 3 + 2];
  const float ge = p.g_entropy ? p.g_entropy[row] : 0.f;
  auto rest_of = [&](float x) {
    const float lp = (x - m) - log_s, pr = __builtin_amdgcn_exp2f(lp * LOG2E);
    return p.g_entropy ? -pr * __builtin_fmaf(ge, fmaxf(lp, -1e4f) + entropy, total) : -pr * total;      // (-inf times its 0 is nothing)
  };
  char* const out = (char*)p.d_logits + row * p.d_stride * SIZE;
  auto put = [&](int64_t e, float y) {
    if constexpr (F32) ((float*)out)[e] = y;
    else ((bf16_t*)out)[e] = (bf16_t)y;
  };
  // Entries with gradients of their own are written by the first output that asks for them, with the others' in their order, and the rest
  // below.  (Entry by entry, each looking through all outputs, 100 tokens of 2000 rows of 10000 took 183 us.)
  const bool dense = asked > 2 * NT;     // (so many that they are worth a list of those that look through the others)
  auto one = [&](int at) { return (several[at / 32] >> (at % 32) & 1u) == 0; };
  for (int c = threadIdx.x; c < asked; c += NT) {
    const int at = c < NT ? mine : c < LIST ? list[c] : place_in(index_of(c));
    if (at < 0) continue;
    if (one(at)) put(e0 + at, rest_of(c < NT ? early : logit_at<F32>(p, row, e0 + at)) + (c < LIST ? gradient[c] : gradient_of(c)));
    else if (dense && c < LIST) queue[atomicAdd(&queued, 1)] = (uint16_t)c;
  }
  if (repeated) {
    if (dense) __syncthreads();
    const int listed = asked < LIST ? (asked + 7) / 8 * 8 : LIST, n = dense ? queued : 0, rest = dense ? LIST : 0;
    for (int i = threadIdx.x; i < n || i - n + rest < asked; i += NT) {
      const int c = i < n ? queue[i] : i - n + rest, at = c < LIST ? list[c] : place_in(index_of(c));
      if (at < 0 || one(at)) continue;
      float own = c < LIST ? gradient[c] : gradient_of(c);
      bool first = true;
      for (int k0 = 0; k0 < listed; k0 += 8) {
        int l[8];
        float g[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) { l[k] = list[k0 + k]; g[k] = gradient[k0 + k]; }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bool met = l[k] == at && k0 + k != c;
          own += met ? g[k] : 0.f;
          first &= !met || k0 + k > c;
        }
      }
      for (int k = LIST; k < asked; ++k) {
        if (k == c || place_in(index_of(k)) != at) continue;
        own += gradient_of(k);
        first &= k > c;
      }
      if (first) put(e0 + at, rest_of(logit_at<F32>(p, row, e0 + at)) + own);
    }
  }
  const bool apart = (((uintptr_t)out ^ (uintptr_t)((const char*)p.logits + row * p.stride * SIZE)) & 15u) != 0;
#pragma unroll
  for (int c = 0; c < VECS; ++c) {
    const int v = v0 + c * NT + threadIdx.x;
    if (c >= p.vecs || v >= r.vectors) continue;
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = rest_of(x[c].at(i));
    const int e = r.first(v), at = (c * NT + threadIdx.x) * N;
    const uint32_t taken = hit[at / 32] >> (at % 32) & ((1u << N) - 1u);
    if (r.whole(v) && !apart && taken == 0) {
      uint4 w;
      if constexpr (F32) w = __builtin_bit_cast(uint4, floatx4{y[0], y[1], y[2], y[3]});
      else w = uint4{pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7])};
      __builtin_nontemporal_store(__builtin_bit_cast(uint4v, w), (uint4v*)(out + (int64_t)e * SIZE));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e + i >= 0 && e + i < p.vocab && !(taken >> i & 1u)) put(e + i, y[i]);
    }
  }
}

struct Split { int nt, vecs, parts; };

// How rows are cut up, by their number and length.
Split split_of(const HstuLogProbsArgs& a) {
  const int64_t n = a.dtype == HSTU_SERVE_FP32 ? 4 : 8, vectors = ((int64_t)a.vocab + n - 1 + n - 1) / n;   // (a row may start anywhere)
  Split s;
  // a wave for short rows where there are enough of them to fill the chip, four waves otherwise: forward and backward of 16000 rows of 2000
  // (bf16) with the 10 largest 27 + 35 us against 62 + 49, of 100 rows 11 + 6 against 7 + 6.  Its 64 maxima bound up to 50 of a row's largest
  // entries well: 100 of them reach the bound, with 60 it is 180.  A row of fewer vectors than entries asked for has no bound: all of its entries
  // are ranked, and past the one wave's list of 256 found bit by bit, where four waves pay for
  // longer: 300 wide with the 50 largest, 1024 rows 49 us against 22, 4096 rows 55 against 62, 16384 rows 201 against 216.
  const bool bounded = a.vocab <= 256 || a.vocab / n >= a.top;
  s.nt = vectors <= 64 * VECS && (a.rows >= (bounded ? 1024 : 4096) ? a.top <= 50 : vectors <= 128 && a.top <= 16) ? 64 : 256;
  int64_t parts = (vectors + (int64_t)s.nt * VECS - 1) / ((int64_t)s.nt * VECS);
  // few rows: more parts, so that they fill the chip, while the join holds all of a row's largest entries at once
  while (a.rows * parts < 256 && parts * s.nt * 2 <= vectors && 2 * parts * a.top <= 2048) parts *= 2;
  s.vecs = (int)((vectors + parts * s.nt - 1) / (parts * s.nt));
  s.parts = (int)((vectors + (int64_t)s.nt * s.vecs - 1) / ((int64_t)s.nt * s.vecs));
  return s;
}

int check(const HstuLogProbsArgs* a) {
  if (!a) return serve_fail(HSTU_SERVE_ERR_NULL, "args is null");
  if (a->struct_size != sizeof(HstuLogProbsArgs) || a->version != HSTU_SERVE_ABI_VERSION)
    return serve_fail(HSTU_SERVE_ERR_VERSION, "struct_size %u version %u, expected %zu and %d", a->struct_size, a->version, sizeof(HstuLogProbsArgs), HSTU_SERVE_ABI_VERSION);
  if (a->dtype != HSTU_SERVE_BF16 && a->dtype != HSTU_SERVE_FP32) return serve_fail(HSTU_SERVE_ERR_SHAPE, "dtype %d", a->dtype);
  // (a thread's next token, and the tokens and the largest entries together, are counted in 32 bits)
  if (a->rows < 0 || a->vocab < 1 || a->vocab > 1 << 30 || a->count < 0 || a->count > 1 << 30) return serve_fail(HSTU_SERVE_ERR_SHAPE, "rows=%lld vocab=%d count=%d (each row's at most 2^30)", (long long)a->rows, a->vocab, a->count);
  if (a->top < 0 || a->top > MAX_TOP || a->top > a->vocab) return serve_fail(HSTU_SERVE_ERR_SHAPE, "top=%d: at most %d and the vocabulary", a->top, MAX_TOP);
  return HSTU_SERVE_OK;
}

size_t part_bytes(const HstuLogProbsArgs& a, const Split& s) {
  return s.parts == 1 ? 0 : (size_t)a.rows * s.parts * (3 * sizeof(float) + (size_t)a.top * (sizeof(float) + sizeof(int32_t)));
}

int fill(const HstuLogProbsArgs* a, const Split& s, Params* p) {
  const size_t size = a->dtype == HSTU_SERVE_FP32 ? 4 : 2;
  if (!a->logits || (a->count > 0 && !a->tokens)) return serve_fail(HSTU_SERVE_ERR_NULL, "logits or tokens is null");
  if ((uintptr_t)a->logits % size) return serve_fail(HSTU_SERVE_ERR_SHAPE, "logits are not aligned to their type");
  if (a->rows > SERVE_THREADS / s.nt / s.parts) return serve_fail(HSTU_SERVE_ERR_SHAPE, "%lld rows of %d parts are too many for one call", (long long)a->rows, s.parts);
  *p = Params{};
  p->logits = a->logits; p->stride = a->stride; p->tokens = a->tokens;
  p->log_probs = a->log_probs; p->entropy = a->entropy; p->stats = a->stats;
  p->top_log_probs = a->top_log_probs; p->top_tokens = a->top_tokens;
  p->rows = a->rows; p->vocab = a->vocab; p->count = a->count; p->top = a->top;
  p->parts = s.parts; p->vecs = s.vecs; p->sums_t = a->entropy != nullptr;
  return HSTU_SERVE_OK;
}

}  // namespace

extern "C" {

size_t hstu_log_probs_workspace_bytes(const HstuLogProbsArgs* a) {
  serve_clear_error();
  if (check(a) || a->rows == 0) return 0;
  return part_bytes(*a, split_of(*a));
}

int hstu_log_probs_fwd(const HstuLogProbsArgs* a, void* stream) {
  serve_clear_error();
  if (const int rc = check(a)) return rc;
  if (a->rows == 0) return HSTU_SERVE_OK;
  const Split s = split_of(*a);
  Params p;
  if (const int rc = fill(a, s, &p)) return rc;
  if ((a->count > 0 && !a->log_probs) || (a->top > 0 && (!a->top_log_probs || !a->top_tokens))) return serve_fail(HSTU_SERVE_ERR_NULL, "an output is null");
  const size_t need = part_bytes(*a, s);
  if (need && (!a->workspace || a->workspace_bytes < need || !serve_aligned16(a->workspace)))
    return serve_fail(HSTU_SERVE_ERR_WORKSPACE, "workspace of %zu bytes on a 16-byte boundary needed, got %zu", need, a->workspace_bytes);
  p.part_stats = (float*)a->workspace;
  p.part_value = p.part_stats + a->rows * s.parts * 3;
  p.part_index = (int32_t*)(p.part_value + a->rows * s.parts * a->top);
  hipStream_t st = (hipStream_t)stream;
  const bool f32 = a->dtype == HSTU_SERVE_FP32;
  const uint32_t grid = (uint32_t)(a->rows * s.parts);
#define PART(F32, NT)                                                              \
  do {                                                                             \
    if (p.top) hstu_log_probs_part<F32, NT, true><<<grid, NT, 0, st>>>(p);         \
    else hstu_log_probs_part<F32, NT, false><<<grid, NT, 0, st>>>(p);              \
  } while (0)
  if (s.nt == 64) { if (f32) PART(true, 64); else PART(false, 64); }
  else { if (f32) PART(true, 256); else PART(false, 256); }
#undef PART
  if (const int rc = serve_launched("hstu_log_probs_part")) return rc;
  if (s.parts > 1) {
    // (a wave where its lanes hold all of a row's parts at once)
    const bool small = s.parts <= 64 && (int64_t)s.parts * a->top <= 256 && a->top <= 64;
    const uint32_t rows = (uint32_t)a->rows;
    if (small) { if (f32) hstu_log_probs_join<true, 64><<<rows, 64, 0, st>>>(p); else hstu_log_probs_join<false, 64><<<rows, 64, 0, st>>>(p); }
    else { if (f32) hstu_log_probs_join<true, 256><<<rows, 256, 0, st>>>(p); else hstu_log_probs_join<false, 256><<<rows, 256, 0, st>>>(p); }
    return serve_launched("hstu_log_probs_join");
  }
  return HSTU_SERVE_OK;
}

int hstu_log_probs_bwd(const HstuLogProbsArgs* a, void* stream) {
  serve_clear_error();
  if (const int rc = check(a)) return rc;
  if (a->rows == 0) return HSTU_SERVE_OK;
  const Split s = split_of(*a);
  Params p;
  if (const int rc = fill(a, s, &p)) return rc;
  const size_t size = a->dtype == HSTU_SERVE_FP32 ? 4 : 2;
  if (!a->stats || !a->d_logits || (a->g_top && !a->top_tokens)) return serve_fail(HSTU_SERVE_ERR_NULL, "stats, d_logits or top_tokens is null");
  if ((uintptr_t)a->d_logits % size) return serve_fail(HSTU_SERVE_ERR_SHAPE, "d_logits is not aligned to its type");
  p.g_tokens = a->count > 0 ? a->g_tokens : nullptr; p.g_entropy = a->g_entropy; p.g_top = a->top > 0 ? a->g_top : nullptr;
  p.d_logits = a->d_logits; p.d_stride = a->d_stride;
  hipStream_t st = (hipStream_t)stream;
  const bool f32 = a->dtype == HSTU_SERVE_FP32;
  const uint32_t grid = (uint32_t)(a->rows * s.parts);
  if (s.nt == 64) {
    if (f32) hstu_log_probs_backward<true, 64><<<grid, 64, 0, st>>>(p);
    else hstu_log_probs_backward<false, 64><<<grid, 64, 0, st>>>(p);
  } else {
    if (f32) hstu_log_probs_backward<true, 256><<<grid, 256, 0, st>>>(p);
    else hstu_log_probs_backward<false, 256><<<grid, 256, 0, st>>>(p);
  }
  return serve_launched("hstu_log_probs_backward");
}

}
