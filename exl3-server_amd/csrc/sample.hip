// The choice of a token from a row of logits with temperature, top-k, top-p and min-p from a
// given random number (gfx950).
//
// A row's order is by logit, largest first, equal ones by index. With t_i = (max - x_i) / T
// and w_i = exp(-t_i), the kept tokens are the shortest of three beginnings of the order:
// the first top_k; of those, as many as it takes to hold top_p of their weight; those with
// w >= min_p (the first token is always kept). The token is the first whose running weight
// exceeds u times the kept weight.
//
// Every weight is taken in f64 and held as an integer of 2^-44 of the largest: sums of
// integers are the same in any order, so the histogram's atomics and the split over
// workgroups change nothing, and a row of 2^19 tokens fits 64 bits. (A weight under 2^-45 of
// the largest counts as 0.) Rows are read in 16-byte pieces, several in flight; a product in
// f32 tells first which tokens can matter, and only those are weighed.
//
//  k_sample_max   grid (split, row): the split's largest logit and its index.
//  k_sample_hist  grid (split, row): counts and weights of the split's tokens in bins of 1/64
//                 of t (2000 bins down to 2^-45), and the count and weight at min_p or above.
//  k_sample_pick  a workgroup per row: the splits' histograms added up and scanned give the
//                 bins in which top-k, top-p and the random number end; only those bins'
//                 tokens are gathered from the row, sorted and summed token by token. A bin
//                 with more tokens than the list holds is narrowed by the logits' bits
//                 (11, 11, 10) with the same histogram.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>
#include <type_traits>

#include "elem.hpp"
#include "exl3_device.hpp"
#include "exl3_internal.hpp"
#include "exl3_moe.h"

using namespace exl3d;
using namespace exl3e;

namespace {

constexpr int kMaxVocab = 1 << 19;
constexpr int kBins = 2048;           // 2000 used
constexpr double kPerT = 64.0;        // bins per unit of t
constexpr double kMaxT = 31.25;       // exp(-31.25) < 2^-45
constexpr double kOne = 17592186044416.0;  // 2^44
constexpr int kThreads = 512;
constexpr int kPickThreads = 1024;
constexpr int kList = 2048;           // tokens of a sorted list
constexpr int kMaxSplits = 16;
static_assert(kMaxSplits <= 64, "a lane per split");
static_assert(kMaxT * kPerT < kBins, "every weighted token has a bin");
static_assert(kList == kBins && kPickThreads * 2 == kBins, "two bins a thread");

typedef unsigned long long u64;

// Logits as keys that order like them (0: NaN; -0 as +0), and back.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0;
  const uint32_t b = bitcast<uint32_t>(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return bitcast<float>(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kMaskedKey = 0x007fffffu;  // the key of -inf; NaN is below it

struct SampleArgs {
  const void *logits;
  int64_t rows, stride;
  int32_t vocab, splits, per_split;
  float temperature, top_p, min_p;
  int32_t top_k;
  const float *temperatures, *top_ps, *min_ps;
  const int32_t *top_ks;
  const float *u;
  int32_t *ids;
  float *probs;
  u64 *best;        // (rows, splits): key << 32 | ~index of the split's first token
  u64 *mass;        // (rows, splits, kBins)
  uint32_t *count;  // (rows, splits, kBins)
  u64 *min_mass;    // (rows, splits): weight at min_p or above
};

__device__ __forceinline__ double temperature_of(const SampleArgs &a, int64_t row) {
  return (double)(a.temperatures ? a.temperatures[row] : a.temperature);
}

// A row's tokens against its largest logit m.
struct Weigher {
  float m;
  double temp, inv;
  __device__ __forceinline__ Weigher(float m, double temp) : m(m), temp(temp), inv(1.0 / temp) {}
  // The logits whose t may lie in [lo, hi], with a margin for the roundings of its ends.
  struct Range {
    float least, most;
    __device__ __forceinline__ bool has(float x) const { return x >= least && x <= most; }
  };
  __device__ __forceinline__ Range range(double lo, double hi) const {
    if (m == INFINITY) return Range{m, m};
    const double least = (double)m - temp * (hi + 1e-3), most = (double)m - temp * (lo - 1e-3);
    return Range{(float)(least - 1e-6 * fabs(least) - 1e-40), (float)(most + 1e-6 * fabs(most) + 1e-40)};
  }
  // t, or one past kMaxT for a token that is never taken.
  __device__ __forceinline__ double t(float x) const {
    if (!(x > -INFINITY)) return 1e300;
    if (x == m) return 0.0;  // also +inf
    const double d = ((double)m - (double)x) * inv;
    return d < 1e300 ? d : 1e300;
  }
  static __device__ __forceinline__ int bin(double t) { return (int)(t * kPerT); }
  // exp(-t) 2^44 for t <= kMaxT: -t = (n + f) ln 2, the series of e^(f ln 2) up to the 11th power
  // (off by 7e-15 of itself).
  static __device__ __forceinline__ double weight(double t) {
    const double y = t * -1.4426950408889634074, n = rint(y), r = (y - n) * 0.69314718055994530942;
    double p = 2.5052108385441719e-8;
    p = fma(p, r, 2.7557319223985891e-7);
    p = fma(p, r, 2.7557319223985893e-6);
    p = fma(p, r, 2.4801587301587302e-5);
    p = fma(p, r, 1.9841269841269841e-4);
    p = fma(p, r, 1.3888888888888889e-3);
    p = fma(p, r, 8.3333333333333333e-3);
    p = fma(p, r, 4.1666666666666667e-2);
    p = fma(p, r, 0.16666666666666667);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n + 44);
  }
  // To the nearest integer: the sum's low bits are it.
  static __device__ __forceinline__ u64 fixed(double w) {
    return bitcast<u64>(w + 4503599627370496.0) & 0x000fffffffffffffull;
  }
};

struct AllValues {
  __device__ __forceinline__ bool has(float) const { return true; }
};

// f(index, value) for the values [first, last) of a row that `wanted` has, by `step` threads of
// which this is thread tid: 16-byte pieces, kAhead of them loaded before the first is taken;
// what is left of a row one by one. Pieces with no wanted value in a whole wave cost
// their comparisons alone.
template <typename E, int kAhead, typename R, typename F>
__device__ __forceinline__ void each_value(const E *row, int first, int last, int tid, int step, const R &wanted, F &&f) {
  constexpr int N = 16 / sizeof(E);
  typedef E piece __attribute__((ext_vector_type(N), aligned(sizeof(E))));
  const int pieces = (last - first) / N;
  for (int p = tid; p < pieces; p += kAhead * step) {
    piece x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      x[k] = *reinterpret_cast<const piece *>(row + first + (int64_t)min(p + k * step, pieces - 1) * N);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      uint32_t which = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) which |= wanted.has(to_f32((E)x[k][i])) ? 1u << i : 0u;
      if (p + k * step >= pieces) which = 0;
      if constexpr (!std::is_same_v<R, AllValues>) {
        // few are wanted: one at a time
        while (which) {
          const int i = __ffs(which) - 1;
          which &= which - 1;
          float v = 0.0f;
#pragma unroll
          for (int n = 0; n < N; ++n) v = n == i ? to_f32((E)x[k][n]) : v;
          f(first + (p + k * step) * N + i, v);
        }
      } else if (which) {
#pragma unroll
        for (int i = 0; i < N; ++i) f(first + (p + k * step) * N + i, to_f32((E)x[k][i]));
      }
    }
  }
  for (int i = first + pieces * N + tid; i < last; i += step) {
    const float v = to_f32(row[i]);
    if (wanted.has(v)) f(i, v);
  }
}

template <typename T, typename Op>
__device__ __forceinline__ T wave_reduce(T v, Op op) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = op(v, (T)__shfl_xor(v, o));
  return v;
}

// The row's first token over its splits.
__device__ __forceinline__ u64 row_best(const SampleArgs &a, int64_t row) {
  const int lane = threadIdx.x & 63;
  u64 b = lane < a.splits ? a.best[row * a.splits + lane] : 0;
  return wave_reduce(b, [](u64 x, u64 y) { return x > y ? x : y; });
}

template <typename E>
__global__ __launch_bounds__(kThreads) void k_sample_max(SampleArgs a) {
  __shared__ u64 red[kThreads / 64];
  const int64_t row = blockIdx.y;
  const int first = blockIdx.x * a.per_split, last = min(a.vocab, first + a.per_split);
  const E *x = reinterpret_cast<const E *>(a.logits) + row * a.stride;
  // (a thread's indices ascend, so the first of equal keys stays)
  uint32_t most = 0;
  int at = first;
  each_value<E, 4>(x, first, last, threadIdx.x, kThreads, AllValues{}, [&](int i, float v) {
    const uint32_t k = key_of(v);
    if (k > most) most = k, at = i;
  });
  u64 b = (u64)most << 32 | (uint32_t)~at;
  b = wave_reduce(b, [](u64 p, u64 q) { return p > q ? p : q; });
  if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = b;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kThreads / 64; ++i) b = red[i] > b ? red[i] : b;
    a.best[row * a.splits + blockIdx.x] = b;
  }
}

template <typename E>
__global__ __launch_bounds__(kThreads) void k_sample_hist(SampleArgs a) {
  __shared__ u64 mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ u64 red[kThreads / 64];
  const int64_t row = blockIdx.y;
  const double temp = temperature_of(a, row);
  const u64 best = row_best(a, row);
  if (!(temp > 0.0) || (uint32_t)(best >> 32) <= kMaskedKey) return;  // the first token, or none
  for (int i = threadIdx.x; i < kBins; i += kThreads) mass[i] = 0, count[i] = 0;
  __syncthreads();
  const Weigher W(of_key((uint32_t)(best >> 32)), temp);
  const double least = kOne * (double)(a.min_ps ? a.min_ps[row] : a.min_p);
  const int first = blockIdx.x * a.per_split, last = min(a.vocab, first + a.per_split);
  const E *x = reinterpret_cast<const E *>(a.logits) + row * a.stride;
  u64 above = 0;
  const Weigher::Range weighed = W.range(0.0, kMaxT);
  each_value<E, 2>(x, first, last, threadIdx.x, kThreads, AllValues{}, [&](int, float v) {
    if (!weighed.has(v)) return;
    const double t = W.t(v);
    if (t >= kMaxT) return;
    const double w = W.weight(t);
    const u64 f = W.fixed(w);
    atomicAdd(&count[W.bin(t)], 1u);
    atomicAdd(&mass[W.bin(t)], f);
    if (!(w < least)) above += f;
  });
  above = wave_reduce(above, [](u64 p, u64 q) { return p + q; });
  if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = above;
  __syncthreads();
  const int64_t at = (row * a.splits + blockIdx.x) * kBins;
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    a.mass[at + i] = mass[i];
    a.count[at + i] = count[i];
  }
  if (threadIdx.x == 0) {
    for (int i = 1; i < kThreads / 64; ++i) above += red[i];
    a.min_mass[row * a.splits + blockIdx.x] = above;
  }
}

// Running sums over two bins a thread: the bins' own values in, the sums up to and with them out.
struct PickShared {
  u64 mass[kBins];
  u64 list[kList];  // ~key << 32 | index, ascending: the order
  uint32_t count[kBins];
  u64 wave_mass[kPickThreads / 64];
  uint32_t wave_count[kPickThreads / 64];
  int found, n;
  u64 before_mass;
  uint32_t before_count;
};

__device__ void scan_bins(PickShared &s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const u64 m0 = s.mass[2 * tid], m1 = s.mass[2 * tid + 1];
  const uint32_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
  u64 m = m0 + m1;
  uint32_t c = c0 + c1;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 pm = __shfl_up(m, o);
    const uint32_t pc = __shfl_up(c, o);
    if (lane >= o) m += pm, c += pc;
  }
  if (lane == 63) s.wave_mass[wave] = m, s.wave_count[wave] = c;
  __syncthreads();
  for (int w = 0; w < wave; ++w) m += s.wave_mass[w], c += s.wave_count[w];
  s.mass[2 * tid + 1] = m;
  s.mass[2 * tid] = m - m1;
  s.count[2 * tid + 1] = c;
  s.count[2 * tid] = c - c1;
  __syncthreads();
}

// What ends a beginning of the order: the first token at which `count` tokens are reached, or
// weight >= / > `mass`.
struct Until {
  enum Kind { kCount, kAtLeast, kMore } kind;
  uint32_t count;
  double mass;
  __device__ __forceinline__ bool met(uint32_t c, u64 m) const {
    return kind == kCount ? c >= count : kind == kAtLeast ? (double)m >= mass : (double)m > mass;
  }
};

// The first of the scanned bins (descending weight) where `u` is met; kBins if none.
__device__ int first_bin(PickShared &s, const Until &u) {
  if (threadIdx.x == 0) s.found = kBins;
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kPickThreads)
    if (u.met(s.count[i], s.mass[i]) && (i == 0 || !u.met(s.count[i - 1], s.mass[i - 1]))) s.found = i;
  __syncthreads();
  const int b = s.found;
  __syncthreads();
  return b;
}

// Sorts s.list[0..n) ascending; n <= kList.
__device__ void sort_list(PickShared &s, int n) {
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kPickThreads) s.list[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j; j >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += kPickThreads) {
        const int p = 2 * i - (i & (j - 1)), q = p + j;
        const u64 x = s.list[p], y = s.list[q];
        if ((x > y) == ((p & k) == 0)) s.list[p] = y, s.list[q] = x;
      }
      __syncthreads();
    }
}

struct Found {
  int32_t id;
  uint32_t key, count;  // its logit, and tokens and weight up to and with it
  u64 mass;
};

template <typename E>
struct Row {
  const E *x;
  int vocab;
  Weigher W;
  // f(index, value, t) for the tokens of bins [b0, b1]
  template <typename F>
  __device__ __forceinline__ void each_in(int b0, int b1, F &&f) const {
    each_value<E, 4>(x, 0, vocab, threadIdx.x, kPickThreads, W.range(b0 / kPerT, (b1 + 1) / kPerT), [&](int i, float v) {
      const double t = W.t(v);
      if (t < kMaxT && W.bin(t) >= b0 && W.bin(t) <= b1) f(i, v, t);
    });
  }
};

// The first token of the sorted list where `u` is met, with `before` in front of the list (the
// last one where rounding leaves none). Every thread gets it.
template <typename E>
__device__ Found in_list(PickShared &s, const Row<E> &row, int n, const Until &u, uint32_t before_count, u64 before_mass) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  u64 own[2], m = 0;
  for (int k = 0; k < 2; ++k) {
    const int i = 2 * tid + k;
    own[k] = i < n ? row.W.fixed(row.W.weight(row.W.t(of_key((uint32_t)~(s.list[i] >> 32))))) : 0;
    m += own[k];
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 pm = __shfl_up(m, o);
    if (lane >= o) m += pm;
  }
  if (lane == 63) s.wave_mass[wave] = m;
  if (tid == 0) s.found = n - 1;
  __syncthreads();
  m += before_mass;
  for (int w = 0; w < wave; ++w) m += s.wave_mass[w];
  const u64 upto[2] = {m - own[1], m};
  for (int k = 0; k < 2; ++k) {
    const int i = 2 * tid + k;
    if (i < n && u.met(before_count + i + 1, upto[k]) && (!u.met(before_count + i, upto[k] - own[k]) || i == 0))
      atomicMin(&s.found, i);
  }
  __syncthreads();
  const int at = s.found;
  if (at / 2 == tid) s.before_mass = upto[at & 1];
  __syncthreads();
  const Found f{(int32_t)(uint32_t)s.list[at], (uint32_t)~(s.list[at] >> 32), before_count + at + 1, s.before_mass};
  __syncthreads();
  return f;
}

// The tokens of bins [b0, b1] into the list, sorted; there are at most kList.
template <typename E>
__device__ int gather(PickShared &s, const Row<E> &row, int b0, int b1) {
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  row.each_in(b0, b1, [&](int i, float v, double) {
    const int at = atomicAdd(&s.n, 1);
    if (at < kList) s.list[at] = (u64)(uint32_t)~key_of(v) << 32 | (uint32_t)i;
  });
  __syncthreads();
  const int n = min(s.n, kList);
  sort_list(s, n);
  return n;
}

// As in_list, over the tokens of one bin of any size: the logits' bits from the top, 11, 11
// and 10 of them, until all tokens left have one logit; of those the index decides. Uses
// s.mass and s.count.
template <typename E>
__device__ Found in_bin(PickShared &s, const Row<E> &row, int bin, const Until &u, uint32_t before_count, u64 before_mass) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0;  // the bits of ~key found so far, in place
  int low = 32;         // bits below them
  for (int round = 0; round < 3; ++round) {
    const int bits = round < 2 ? 11 : 10, next = low - bits;
    for (int i = tid; i < kBins; i += kPickThreads) s.mass[i] = 0, s.count[i] = 0;
    __syncthreads();
    row.each_in(bin, bin, [&](int, float v, double t) {
      const uint32_t c = ~key_of(v);
      if (low < 32 && (c ^ prefix) >> low) return;
      const int at = (c >> next) & ((1 << bits) - 1);
      atomicAdd(&s.count[at], 1u);
      atomicAdd(&s.mass[at], Weigher::fixed(Weigher::weight(t)));
    });
    __syncthreads();
    scan_bins(s);
    const Until here{u.kind, u.kind == Until::kCount ? u.count - before_count : 0, u.mass};
    if (tid == 0) s.found = kBins;
    __syncthreads();
    const uint32_t all = s.count[kBins - 1];
    for (int i = tid; i < kBins; i += kPickThreads) {
      const uint32_t c0 = i ? s.count[i - 1] : 0;
      if (s.count[i] > c0 && (here.met(s.count[i], before_mass + s.mass[i]) || s.count[i] == all)) atomicMin(&s.found, i);
    }
    __syncthreads();
    const int at = s.found;
    before_count += at ? s.count[at - 1] : 0;
    before_mass += at ? s.mass[at - 1] : 0;
    prefix |= (uint32_t)at << next;
    low = next;
    __syncthreads();
  }
  // ties: how many of this logit it takes, and which index that is
  const uint32_t key = ~prefix;
  const float logit = of_key(key);
  const u64 w = Weigher::fixed(Weigher::weight(row.W.t(logit)));
  uint32_t ties = 0;
  {
    u64 c = 0;
    each_value<E, 4>(row.x, 0, row.vocab, tid, kPickThreads, AllValues{}, [&](int, float v) { c += v == logit; });
    c = wave_reduce(c, [](u64 p, u64 q) { return p + q; });
    if ((tid & 63) == 0) s.wave_count[tid >> 6] = (uint32_t)c;
    __syncthreads();
    for (int i = 0; i < kPickThreads / 64; ++i) ties += s.wave_count[i];
    __syncthreads();
  }
  uint32_t lo = 1, hi = ties;  // the least n for which before + n of them meet `u`
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (u.met(before_count + mid, before_mass + mid * w)) hi = mid;
    else lo = mid + 1;
  }
  // the lo-th index with this logit: pieces of the row in index order
  if (tid == 0) s.found = 0;
  uint32_t seen = 0;
  for (int base = 0; base < row.vocab; base += kPickThreads) {
    const int i = base + tid;
    const bool hit = i < row.vocab && to_f32(row.x[i]) == logit;
    const u64 votes = __ballot(hit);
    if ((tid & 63) == 0) s.wave_count[tid >> 6] = __popcll(votes);
    __syncthreads();
    uint32_t mine = seen + __popcll(votes & ((2ull << (tid & 63)) - 1)), total = seen;
    for (int v = 0; v < kPickThreads / 64; ++v) {
      if (v < (tid >> 6)) mine += s.wave_count[v];
      total += s.wave_count[v];
    }
    if (hit && mine == lo) s.found = i;
    __syncthreads();
    seen = total;
    if (seen >= lo) break;
  }
  const Found f{s.found, key, before_count + lo, before_mass + lo * w};
  __syncthreads();
  return f;
}

template <typename E>
__global__ __launch_bounds__(kPickThreads) void k_sample_pick(SampleArgs a) {
  __shared__ PickShared s;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  const u64 best = row_best(a, r);
  const double temp = temperature_of(a, r);
  const bool none = (uint32_t)(best >> 32) <= kMaskedKey;
  if (none || !(temp > 0.0)) {
    if (tid == 0) {
      a.ids[r] = none ? -1 : (int32_t)~(uint32_t)best;
      if (a.probs) a.probs[r] = none ? 0.0f : 1.0f;
    }
    return;
  }
  const Row<E> row{reinterpret_cast<const E *>(a.logits) + r * a.stride, a.vocab,
                   Weigher(of_key((uint32_t)(best >> 32)), temp)};
  // bins of the whole row, added up from its splits and scanned
  auto whole_row = [&] {
    for (int i = tid; i < kBins; i += kPickThreads) {
      u64 m = 0;
      uint32_t c = 0;
#pragma unroll 8
      for (int k = 0; k < a.splits; ++k) {
        m += a.mass[(r * a.splits + k) * kBins + i];
        c += a.count[(r * a.splits + k) * kBins + i];
      }
      s.mass[i] = m;
      s.count[i] = c;
    }
    __syncthreads();
    scan_bins(s);
  };
  whole_row();
  int listed = 0, list_from = 1, list_to = 0;  // the list holds bins [list_from, list_to]
  // The first token where `u` is met, or the last of all if none is.
  auto find = [&](const Until &u) -> Found {
    int b = first_bin(s, u);
    if (b == kBins) b = first_bin(s, Until{Until::kCount, s.count[kBins - 1], 0.0});
    auto before = [&](int x) { return x ? s.count[x - 1] : 0u; };
    if (b < list_from || b > list_to) {
      list_from = s.count[b] <= (uint32_t)kList ? 0 : b;
      list_to = b;
      if (s.count[b] - before(list_from) > (uint32_t)kList) {
        const uint32_t c = before(b);
        const u64 m = b ? s.mass[b - 1] : 0;
        list_from = 1, list_to = 0;
        __syncthreads();
        const Found f = in_bin(s, row, b, u, c, m);
        whole_row();
        return f;
      }
      listed = gather(s, row, list_from, list_to);
    }
    return in_list(s, row, listed, u, before(list_from), list_from ? s.mass[list_from - 1] : 0);
  };
  u64 kept = s.mass[kBins - 1];
  const int32_t top_k = a.top_ks ? a.top_ks[r] : a.top_k;
  if (top_k > 0 && (uint32_t)top_k < s.count[kBins - 1]) kept = find(Until{Until::kCount, (uint32_t)top_k, 0.0}).mass;
  const float top_p = a.top_ps ? a.top_ps[r] : a.top_p;
  if (top_p < 1.0f) kept = find(Until{Until::kAtLeast, 0, (double)top_p * (double)kept}).mass;
  u64 above = tid % 64 < a.splits ? a.min_mass[r * a.splits + tid % 64] : 0;
  above = wave_reduce(above, [](u64 p, u64 q) { return p + q; });
  const u64 first = (u64)kOne;
  above = above < first ? first : above;
  kept = above < kept ? above : kept;
  const float u = a.u[r];
  // the last kept token where u is 1 or more (or rounding would pass it), the first where u is negative or NaN
  double goal = (u > 0.0f ? (double)u : 0.0) * (double)kept;
  const Found f = goal < (double)kept ? find(Until{Until::kMore, 0, goal}) : find(Until{Until::kAtLeast, 0, (double)kept});
  if (tid == 0) {
    a.ids[r] = f.id;
    if (a.probs) a.probs[r] = (float)(exp(-row.W.t(of_key(f.key))) / ((double)kept / kOne));
  }
}

// Tokens per split: at least 2048, so that the histograms cost less than the row.
int splits_of(int64_t rows, int64_t vocab) {
  int64_t n = (vocab + 2047) / 2048;
  const int64_t enough = (2048 + rows - 1) / rows;  // 8 workgroups a CU
  n = n < enough ? n : enough;
  return (int)(n < 1 ? 1 : n > kMaxSplits ? kMaxSplits : n);
}

struct SampleWs {
  size_t best, mass, count, min_mass, total;
};

SampleWs sample_ws(int64_t rows, int64_t vocab) {
  const size_t n = (size_t)rows * splits_of(rows, vocab);
  SampleWs w;
  w.best = 0;
  w.min_mass = exl3h::align_up(n * 8, 256);
  w.mass = w.min_mass + exl3h::align_up(n * 8, 256);
  w.count = w.mass + n * kBins * 8;
  w.total = w.count + n * kBins * 4;
  return w;
}

bool bad_shape(int64_t rows, int64_t vocab) { return rows < 0 || rows > 65535 || vocab < 1 || vocab > kMaxVocab; }

}  // namespace

using namespace exl3h;

extern "C" {

size_t exl3_sample_workspace_size(int64_t rows, int64_t vocab) {
  return bad_shape(rows, vocab) || rows == 0 ? 0 : sample_ws(rows, vocab).total;
}

exl3_status exl3_sample(const exl3_sample_config *cfg, const void *logits, int64_t rows, int64_t vocab,
                        int64_t row_stride, const float *u, int32_t *ids, float *probs, void *workspace,
                        size_t workspace_bytes, exl3_stream_t stream) {
  if (!cfg) return fail(EXL3_ERR_INVALID, "exl3_sample: null config");
  if (cfg->dtype != EXL3_ST_F16 && cfg->dtype != EXL3_ST_BF16 && cfg->dtype != EXL3_ST_F32)
    return fail(EXL3_ERR_UNSUPPORTED, "exl3_sample: logits must be f16, bf16 or f32");
  if (bad_shape(rows, vocab))
    return fail(EXL3_ERR_INVALID, "exl3_sample: bad shape (at most 65,535 rows of 1 to 524,288 logits)");
  if (row_stride < vocab || row_stride > ((int64_t)1 << 40))
    return fail(EXL3_ERR_INVALID, "exl3_sample: the row stride must be at least the vocabulary");
  if (rows == 0) return EXL3_OK;
  if (!logits || !u || !ids) return fail(EXL3_ERR_INVALID, "exl3_sample: null argument");
  const uintptr_t size = cfg->dtype == EXL3_ST_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size ||
      (reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(probs) |
       reinterpret_cast<uintptr_t>(cfg->temperatures) | reinterpret_cast<uintptr_t>(cfg->top_ks) |
       reinterpret_cast<uintptr_t>(cfg->top_ps) | reinterpret_cast<uintptr_t>(cfg->min_ps)) % 4)
    return fail(EXL3_ERR_INVALID, "exl3_sample: an argument is not aligned to its type");
  const SampleWs w = sample_ws(rows, vocab);
  if (!workspace || workspace_bytes < w.total)
    return fail(EXL3_ERR_WORKSPACE, "exl3_sample: workspace too small: need " + std::to_string(w.total) + " bytes");
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(EXL3_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  SampleArgs a = {};
  a.logits = logits;
  a.rows = rows;
  a.stride = row_stride;
  a.vocab = (int32_t)vocab;
  a.splits = splits_of(rows, vocab);
  a.per_split = (int32_t)((vocab + a.splits - 1) / a.splits);
  a.temperature = cfg->temperature;
  a.top_k = cfg->top_k;
  a.top_p = cfg->top_p;
  a.min_p = cfg->min_p;
  a.temperatures = cfg->temperatures;
  a.top_ks = cfg->top_ks;
  a.top_ps = cfg->top_ps;
  a.min_ps = cfg->min_ps;
  a.u = u;
  a.ids = ids;
  a.probs = probs;
  char *ws = reinterpret_cast<char *>(workspace);
  a.best = reinterpret_cast<u64 *>(ws + w.best);
  a.min_mass = reinterpret_cast<u64 *>(ws + w.min_mass);
  a.mass = reinterpret_cast<u64 *>(ws + w.mass);
  a.count = reinterpret_cast<uint32_t *>(ws + w.count);
  auto go = [&](auto e) {
    using E = decltype(e);
    const dim3 grid((unsigned)a.splits, (unsigned)rows);
    const hipStream_t st = stream_of(stream);
    k_sample_max<E><<<grid, kThreads, 0, st>>>(a);
    if (cfg->temperatures || cfg->temperature > 0.0f) k_sample_hist<E><<<grid, kThreads, 0, st>>>(a);
    k_sample_pick<E><<<(unsigned)rows, kPickThreads, 0, st>>>(a);
  };
  if (cfg->dtype == EXL3_ST_F32) go(float{});
  else with_elem16(cfg->dtype, go);
  EXL3_LAUNCHED("k_sample");
  return EXL3_OK;
}

}  // extern "C"
