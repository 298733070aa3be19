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
//                 of t (2000 bins down to 2^-45) and in groups of 32 bins, the tokens' indices
//                 in the bins' order, and the weight at min_p or above.
//  k_sample_pick  a workgroup per row, for each end of a beginning (top-k, top-p, the random
//                 number): the group it falls in, the bin of the group, the bin's tokens by way
//                 of the splits' index lists, and their order; only those tokens' logits are
//                 read again. A bin with more tokens than the list holds is narrowed by their
//                 logits' and indices' bits, 11 at a time.
// Bound by the histogram's vector instructions for many tokens (64 rows of 154,880 in f32: 8 + 24 +
// 14 us, where reading them once takes 8; its 9.5e6 instructions are about 15 of the 24), and by
// the third kernel's chain of dependent loads for few rows (one row: 3 + 7 + 14 us; the groups, a bin's tokens and their
// logits are three of them for each end). Before the index lists, with the row gathered and
// sorted for each end, one row took 41 us and 8 rows 70.
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
constexpr int kGroups = 64, kInGroup = kBins / kGroups;
constexpr int kList = 1024;           // tokens ordered at once
constexpr int kMaxSplits = 64, kPerSplit = 12288;  // a lane per split; 16-bit places
constexpr float kMost = 3.40282347e38f, kPastBins = (float)(kMaxT * kPerT);
static_assert(kMaxT * kPerT < kBins, "every weighted token has a bin");
constexpr int kMassWords = kPerSplit / 4 > kBins ? kPerSplit / 4 : kBins;
static_assert(kMaxSplits * kPerSplit >= kMaxVocab, "the splits hold any row");
static_assert(kThreads * 4 == kBins && kInGroup == 32, "four bins a thread, eight threads a group");

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
  // for each row and split
  u64 *best;            // key << 32 | ~index of the first token
  u64 *min_mass;        // weight at min_p or above
  u64 *mass;            // (kBins)
  uint32_t *place;      // (kBins): where a bin's indices begin, << 16 | their count
  u64 *group_mass;      // (kGroups)
  uint32_t *group_count;
  uint16_t *order;      // (per_split): indices in the split, by bin
};

__device__ __forceinline__ double temperature_of(const SampleArgs &a, int64_t row) {
  return (double)(a.temperatures ? a.temperatures[row] : a.temperature);
}

// A row's tokens against its largest logit m (never -inf).
struct Weigher {
  float m, half_m, per;  // per: bins per half a logit
  double top, inv, turn; // m (or the largest finite value), 1 / T, 1 / (T ln 2)
  double c[10] = {kOne * 7.072578320978871e-09, kOne * 1.0208693139320117e-07, kOne * 1.3215442682805318e-06,
                  kOne * 1.525265724710113e-05, kOne * 0.00015403530441399083, kOne * 0.0013333558230182842,
                  kOne * 0.009618129107607343,  kOne * 0.05550410866444765,    kOne * 0.24022650695910097,
                  kOne * 0.69314718055995};  // of 2^44 2^f, the highest power first
  __device__ __forceinline__ Weigher(float m, double temp)
      : m(m), half_m(0.5f * m), per((float)(2.0 * kPerT / temp)), top(finite(m)), inv(1.0 / temp),
        turn(1.4426950408889634074 * (1.0 / temp)) {
    // in scalar registers: from vector ones each would be copied for every value (a fused
    // multiply-add overwrites its addend there)
#pragma unroll
    for (int i = 0; i < 10; ++i) asm("" : "+s"(c[i]));
  }
  static __device__ __forceinline__ double finite(float x) { return (double)__builtin_amdgcn_fmed3f(x, -INFINITY, kMost); }
  // The token's bin as a number, by f32 alone (it only has to ascend as the logit falls; halved so
  // that no difference overflows); not under kPastBins for tokens that are never taken.
  __device__ __forceinline__ float place(float x) const {
    const float b = fmaf(-0.5f, x, half_m) * per;
    return x == m ? 0.0f : b;  // (also +inf)
  }
  // exp(-t) 2^44 of a token that has a bin: 2^y = 2^n 2^f with f in [-1/2, 1/2], the latter by the
  // polynomial of degree 10 through 11 Chebyshev points (off by 5e-16 of itself; exact at 0).
  __device__ __forceinline__ double weight(float x) const {
    const double y = (finite(x) - top) * turn, n = rint(y), f = y - n;
    double p = c[0];
#pragma unroll
    for (int i = 1; i < 10; ++i) p = fma(p, f, c[i]);
    p = fma(p, f, kOne);
    return ldexp(p, (int)n);
  }
  // To the nearest integer: the sum's low bits are it.
  static __device__ __forceinline__ u64 fixed(double w) {
    return bitcast<u64>(w + 4503599627370496.0) & 0x000fffffffffffffull;
  }
  // exp(-t).
  __device__ __forceinline__ double share(float x) const { return exp((finite(x) - top) * inv); }
};

// f(index, value) for the values [first, last) of a row, by `step` threads of which this is
// thread tid: 16-byte pieces, kAhead of them loaded before the first is taken; what is left
// of a row one by one. A thread's indices ascend.
template <typename E, int kAhead, typename F>
__device__ __forceinline__ void each_value(const E *row, int first, int last, int tid, int step, F &&f) {
  constexpr int N = 16 / sizeof(E);
  typedef E piece __attribute__((ext_vector_type(N), aligned(sizeof(E))));
  const int pieces = (last - first) / N;
  for (int p = tid; p < pieces; p += kAhead * step) {
    piece x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      x[k] = *reinterpret_cast<const piece *>(row + first + (int64_t)min(p + k * step, pieces - 1) * N);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (p + k * step < pieces)
#pragma unroll
        for (int i = 0; i < N; ++i) f(first + (p + k * step) * N + i, to_f32((E)x[k][i]));
  }
  for (int i = first + pieces * N + tid; i < last; i += step) f(i, to_f32(row[i]));
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
  const int first = min(a.vocab, (int)blockIdx.x * a.per_split), last = min(a.vocab, first + a.per_split);
  const E *x = reinterpret_cast<const E *>(a.logits) + row * a.stride;
  // (the first of equal keys stays)
  uint32_t most = 0;
  int at = first;
  each_value<E, 4>(x, first, last, threadIdx.x, kThreads, [&](int i, float v) {
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
  __shared__ u64 mass[kMassWords];  // then the ordered indices
  __shared__ uint32_t count[kBins];
  __shared__ u64 red[kThreads / 64];
  __shared__ uint32_t wave_count[kThreads / 64];
  const int64_t row = blockIdx.y;
  const double temp = temperature_of(a, row);
  const u64 best = row_best(a, row);
  if (!(temp > 0.0) || (uint32_t)(best >> 32) <= kMaskedKey) return;  // the first token, or none
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < kBins; i += kThreads) mass[i] = 0, count[i] = 0;
  __syncthreads();
  const Weigher W(of_key((uint32_t)(best >> 32)), temp);
  const double least = kOne * (double)(a.min_ps ? a.min_ps[row] : a.min_p);
  const bool weigh_above = least > 0.0;
  const int first = min(a.vocab, (int)blockIdx.x * a.per_split), last = min(a.vocab, first + a.per_split);
  const E *x = reinterpret_cast<const E *>(a.logits) + row * a.stride;
  u64 above = 0;
  each_value<E, 2>(x, first, last, tid, kThreads, [&](int, float v) {
    const float b = W.place(v);
    if (!(b < kPastBins)) return;  // (so for NaN)
    const double w = W.weight(v);
    const u64 f = W.fixed(w);
    atomicAdd(&count[(int)b], 1u);
    atomicAdd(&mass[(int)b], f);
    if (weigh_above) above += w < least ? 0 : f;
  });
  above = wave_reduce(above, [](u64 p, u64 q) { return p + q; });
  if (lane == 0) red[wave] = above;
  __syncthreads();
  // this thread's four bins, and where they begin among the split's tokens
  uint32_t c[4], upto = 0;
  u64 m[4], sum = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    c[k] = count[4 * tid + k];
    m[k] = mass[4 * tid + k];
    upto += c[k];
    sum += m[k];
  }
  const uint32_t own = upto;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t v = __shfl_up(upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 63) wave_count[wave] = upto;
  __syncthreads();
  for (int w = 0; w < wave; ++w) upto += wave_count[w];
  const int64_t split = row * a.splits + blockIdx.x;
  uint32_t begin = upto - own, group = own;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    a.mass[split * kBins + 4 * tid + k] = m[k];
    a.place[split * kBins + 4 * tid + k] = begin << 16 | c[k];
    count[4 * tid + k] = begin;
    begin += c[k];
  }
#pragma unroll
  for (int o = 1; o < kInGroup / 4; o <<= 1) {
    sum += __shfl_xor(sum, o);
    group += __shfl_xor(group, o);
  }
  if (tid % (kInGroup / 4) == 0) {
    a.group_mass[split * kGroups + tid / (kInGroup / 4)] = sum;
    a.group_count[split * kGroups + tid / (kInGroup / 4)] = group;
  }
  if (tid == 0) {
    for (int i = 1; i < kThreads / 64; ++i) above += red[i];
    a.min_mass[split] = above;
  }
  __syncthreads();
  // the indices in the bins' order (within a bin in any), where the weights were: the bins are
  // taken from the logits again, which costs less than the LDS to keep them (3 workgroups a CU)
  uint16_t *ordered = reinterpret_cast<uint16_t *>(mass);
  each_value<E, 2>(x, first, last, tid, kThreads, [&](int i, float v) {
    const float b = W.place(v);
    if (b < kPastBins) ordered[atomicAdd(&count[(int)b], 1u)] = (uint16_t)(i - first);
  });
  __syncthreads();
  uint32_t all = 0;
  for (int w = 0; w < kThreads / 64; ++w) all += wave_count[w];
  uint32_t *to = reinterpret_cast<uint32_t *>(a.order + split * a.per_split);
  for (uint32_t i = tid; 2 * i < all; i += kThreads) to[i] = reinterpret_cast<const uint32_t *>(ordered)[i];
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

// A token's place in the order as a number: ~key (32 bits), index (22 bits).
__device__ __forceinline__ u64 rank_of(uint32_t key, int index) { return (u64)(uint32_t)~key << 22 | (uint32_t)index; }
__device__ __forceinline__ uint32_t rank_key(u64 r) { return (uint32_t)~(r >> 22); }
__device__ __forceinline__ int rank_index(u64 r) { return (int)(r & 0x3fffff); }

struct Found {
  u64 rank, mass;  // the token, and the weight up to and with it
};

struct Item {
  u64 rank, mass;
};

struct PickShared {
  Item list[kList];
  u64 mass[kBins];       // of the buckets of a bin too large for the list
  uint32_t count[kBins];
  uint32_t place[kMaxSplits][kInGroup];
  u64 group_mass[kGroups], bin_mass[kInGroup];
  uint32_t group_count[kGroups], bin_count[kInGroup];
  uint32_t upto[kMaxSplits], begin[kMaxSplits];  // of the bin's tokens, by split
  u64 wave_mass[kThreads / 64];
  uint32_t wave_count[kThreads / 64];
  Found found;
  uint32_t bucket;
};

// Inclusive sums over a wave's first `n` lanes.
__device__ __forceinline__ void wave_scan(int n, uint32_t &c, u64 &m) {
  const int lane = threadIdx.x & 63;
  for (int o = 1; o < n; o <<= 1) {
    const uint32_t pc = __shfl_up(c, o);
    const u64 pm = __shfl_up(m, o);
    if (lane >= o) c += pc, m += pm;
  }
}

template <typename E>
struct Pick {
  const SampleArgs &a;
  PickShared &s;
  const int64_t row;
  const E *x;
  const Weigher W;
  uint32_t upto_count;  // this lane's group: tokens and weight up to and with it
  u64 upto_mass;

  // (c, m): this thread's share of group tid % kGroups
  __device__ Pick(const SampleArgs &a, PickShared &s, int64_t row, const Weigher &W, uint32_t c, u64 m)
      : a(a), s(s), row(row), x(reinterpret_cast<const E *>(a.logits) + row * a.stride), W(W) {
    const int tid = threadIdx.x, lane = tid & 63;
    if (tid < kGroups) s.group_mass[tid] = 0, s.group_count[tid] = 0;
    __syncthreads();
    atomicAdd(&s.group_mass[lane], m);
    atomicAdd(&s.group_count[lane], c);
    __syncthreads();
    upto_mass = s.group_mass[lane];
    upto_count = s.group_count[lane];
    wave_scan(kGroups, upto_count, upto_mass);
  }
  __device__ __forceinline__ uint32_t tokens() const { return __shfl(upto_count, 63); }
  __device__ __forceinline__ u64 weight() const { return __shfl(upto_mass, 63); }

  // The j-th of the bin's tokens (by split, in a split in any order).
  __device__ __forceinline__ int token(uint32_t j) const {
    int k = 0;
#pragma unroll
    for (int o = kMaxSplits / 2; o; o >>= 1)
      if (s.upto[k + o - 1] <= j) k += o;
    const uint32_t at = s.begin[k] + j - (k ? s.upto[k - 1] : 0u);
    return k * a.per_split + a.order[(row * a.splits + k) * a.per_split + at];
  }
  __device__ __forceinline__ u64 mass_of(float v) const { return W.fixed(W.weight(v)); }

  // The first token of the order where `u` is met, or the last of all where none is. Called
  // by the whole workgroup, and the same for all of it.
  __device__ Found find(const Until &u) {
    const int tid = threadIdx.x, lane = tid & 63;
    // its group of bins
    u64 votes = __ballot(u.met(upto_count, upto_mass));
    if (!votes) votes = __ballot(upto_count == tokens());
    const int g = __ffsll(votes) - 1;
    uint32_t before_count = g ? __shfl(upto_count, g - 1) : 0;
    u64 before_mass = g ? __shfl(upto_mass, g - 1) : 0;
    // its bin
    __syncthreads();
    if (tid < kInGroup) s.bin_mass[tid] = 0, s.bin_count[tid] = 0;
    __syncthreads();
    {
      const int b = tid % kInGroup;
      u64 m = 0;
      uint32_t c = 0;
#pragma unroll 4
      for (int k = tid / kInGroup; k < a.splits; k += kThreads / kInGroup) {
        const int64_t at = (row * a.splits + k) * kBins + g * kInGroup + b;
        const uint32_t place = a.place[at];
        m += a.mass[at];
        c += place & 0xffff;
        s.place[k][b] = place;
      }
      atomicAdd(&s.bin_mass[b], m);
      atomicAdd(&s.bin_count[b], c);
    }
    __syncthreads();
    uint32_t c = lane < kInGroup ? s.bin_count[lane] : 0;
    u64 m = lane < kInGroup ? s.bin_mass[lane] : 0;
    wave_scan(kInGroup, c, m);
    votes = __ballot(lane < kInGroup && u.met(before_count + c, before_mass + m));
    if (!votes) votes = __ballot(lane < kInGroup && c == __shfl(c, kInGroup - 1));
    const int b = __ffsll(votes) - 1;
    const uint32_t n = s.bin_count[b];
    before_count += __shfl(c, b) - n;
    before_mass += __shfl(m, b) - s.bin_mass[b];
    // its tokens
    const uint32_t place = lane < a.splits ? s.place[lane][b] : 0;
    uint32_t upto = place & 0xffff;
#pragma unroll
    for (int o = 1; o < kMaxSplits; o <<= 1) {
      const uint32_t v = __shfl_up(upto, o);
      if (lane >= o) upto += v;
    }
    if (tid < kMaxSplits) s.upto[tid] = upto, s.begin[tid] = place >> 16;
    __syncthreads();
    return n <= (uint32_t)kList ? in_list(u, n, before_count, before_mass) : in_buckets(u, n, before_count, before_mass);
  }

  // Few: each token against all of them.
  __device__ Found in_list(const Until &u, uint32_t n, uint32_t before_count, u64 before_mass) {
    for (uint32_t j = threadIdx.x; j < n; j += kThreads) {
      const int i = token(j);
      const float v = to_f32(x[i]);
      s.list[j] = Item{rank_of(key_of(v), i), mass_of(v)};
    }
    __syncthreads();
    // as many lanes an item as there are threads for it (a power of two, in one wave)
    int lanes = 64;
    while (lanes > 1 && (uint32_t)lanes * n > (uint32_t)kThreads) lanes >>= 1;
    for (uint32_t j = threadIdx.x / lanes; j < n; j += kThreads / lanes) {
      const Item own = s.list[j];
      uint32_t c = 0;
      u64 m = 0;
#pragma unroll 4
      for (uint32_t k = threadIdx.x % lanes; k < n; k += lanes) {
        const Item o = s.list[k];
        const bool first = o.rank < own.rank;
        c += first ? 1 : 0;
        m += first ? o.mass : 0;
      }
      for (int o = 1; o < lanes; o <<= 1) {
        c += __shfl_xor(c, o);
        m += __shfl_xor(m, o);
      }
      c += before_count;
      m += before_mass;
      if ((u.met(c + 1, m + own.mass) || c + 1 == before_count + n) && (c == before_count || !u.met(c, m)))
        s.found = Found{own.rank, m + own.mass};
    }
    __syncthreads();
    return s.found;
  }

  // Many: the ranks' bits from the top, 11 at a time, in buckets that are counted and weighed.
  __device__ Found in_buckets(const Until &u, uint32_t n, uint32_t before_count, u64 before_mass) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    u64 prefix = 0;
    for (int low = 44; low >= 0; low -= 11) {
      for (int i = tid; i < kBins; i += kThreads) s.mass[i] = 0, s.count[i] = 0;
      if (tid == 0) s.bucket = kBins;
      __syncthreads();
      for (uint32_t j = tid; j < n; j += kThreads) {
        const int i = token(j);
        const float v = to_f32(x[i]);
        const u64 r = rank_of(key_of(v), i);
        if ((r ^ prefix) >> (low + 11)) continue;
        const int at = (int)(r >> low) & (kBins - 1);
        atomicAdd(&s.count[at], 1u);
        atomicAdd(&s.mass[at], mass_of(v));
      }
      __syncthreads();
      // running sums, four buckets a thread
      uint32_t c[4], cs = 0;
      u64 m[4], ms = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        cs += s.count[4 * tid + k];
        ms += s.mass[4 * tid + k];
        c[k] = cs;
        m[k] = ms;
      }
      const uint32_t c_own = cs;
      const u64 m_own = ms;
      wave_scan(64, cs, ms);
      if (lane == 63) s.wave_count[wave] = cs, s.wave_mass[wave] = ms;
      __syncthreads();
      uint32_t all = 0;
      for (int w = 0; w < kThreads / 64; ++w) {
        if (w < wave) cs += s.wave_count[w], ms += s.wave_mass[w];
        all += s.wave_count[w];
      }
      cs += before_count - c_own;
      ms += before_mass - m_own;
#pragma unroll
      for (int k = 3; k >= 0; --k)
        if (s.count[4 * tid + k] && (u.met(cs + c[k], ms + m[k]) || cs + c[k] == before_count + all))
          atomicMin(&s.bucket, 4u * tid + k);
      __syncthreads();
      const uint32_t at = s.bucket;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at == 4u * tid + k) s.found = Found{cs + c[k] - s.count[at], ms + m[k] - s.mass[at]};  // what is before it
      __syncthreads();
      before_count = (uint32_t)s.found.rank;
      before_mass = s.found.mass;
      prefix |= (u64)at << low;
      if (low == 0) before_mass += s.mass[at];
      __syncthreads();
    }
    return Found{prefix, before_mass};
  }
};

template <typename E>
__global__ __launch_bounds__(kThreads) void k_sample_pick(SampleArgs a) {
  __shared__ PickShared s;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  // everything that needs no other value first: a load that waits for one costs a microsecond
  const int lane = tid & 63;
  u64 best = lane < a.splits ? a.best[r * a.splits + lane] : 0;
  u64 above = lane < a.splits ? a.min_mass[r * a.splits + lane] : 0;
  const double temp = temperature_of(a, r);
  const int32_t top_k = a.top_ks ? a.top_ks[r] : a.top_k;
  const float top_p = a.top_ps ? a.top_ps[r] : a.top_p;
  const float min_p = a.min_ps ? a.min_ps[r] : a.min_p;
  const float u = a.u[r];
  u64 m[kMaxSplits * 64 / kThreads];
  uint32_t c[kMaxSplits * 64 / kThreads];
#pragma unroll
  for (int k = 0; k < kMaxSplits * 64 / kThreads; ++k) {
    const int split = k * (kThreads / 64) + (tid >> 6);
    const int64_t at = (r * a.splits + min(split, a.splits - 1)) * kGroups + lane;
    m[k] = split < a.splits ? a.group_mass[at] : 0;
    c[k] = split < a.splits ? a.group_count[at] : 0;
  }
  best = wave_reduce(best, [](u64 p, u64 q) { return p > q ? p : q; });
  const bool none = (uint32_t)(best >> 32) <= kMaskedKey;
  if (none || !(temp > 0.0)) {
    if (tid == 0) {
      a.ids[r] = none ? -1 : (int32_t)~(uint32_t)best;
      if (a.probs) a.probs[r] = none ? 0.0f : 1.0f;
    }
    return;
  }
#pragma unroll
  for (int k = 1; k < kMaxSplits * 64 / kThreads; ++k) m[0] += m[k], c[0] += c[k];
  Pick<E> pick(a, s, r, Weigher(of_key((uint32_t)(best >> 32)), temp), c[0], m[0]);
  u64 kept = pick.weight();
  if (top_k > 0 && (uint32_t)top_k < pick.tokens()) kept = pick.find(Until{Until::kCount, (uint32_t)top_k, 0.0}).mass;
  if (top_p < 1.0f) kept = pick.find(Until{Until::kAtLeast, 0, (double)top_p * (double)kept}).mass;
  if (min_p > 0.0f) {
    above = wave_reduce(above, [](u64 p, u64 q) { return p + q; });
    const u64 first = (u64)kOne;
    above = above < first ? first : above;
    kept = above < kept ? above : kept;
  }
  // the last kept token where u is 1 or more (or rounding would pass it), the first where u is negative or NaN
  const double goal = (u > 0.0f ? (double)u : 0.0) * (double)kept;
  const Found f = pick.find(goal < (double)kept ? Until{Until::kMore, 0, goal} : Until{Until::kAtLeast, 0, (double)kept});
  if (tid == 0) {
    a.ids[r] = rank_index(f.rank);
    if (a.probs) a.probs[r] = (float)(pick.W.share(of_key(rank_key(f.rank))) / ((double)kept / kOne));
  }
}

// The splits of a row: of at most kPerSplit tokens, more of them where there are few rows, and
// where it can be no more workgroups than the 1024 that the card holds at once (4 a CU): 200
// rows of 32,003 in 5 splits 33.0 us and in 6 35.6, 64 rows of 154,880 in 16 44.9 and in 19 46.5.
struct Split {
  int splits, per_split;
};
Split split_of(int64_t rows, int64_t vocab) {
  const int64_t least = (vocab + kPerSplit - 1) / kPerSplit, most = (vocab + 2047) / 2048;
  int64_t n = 1024 / rows;
  n = n > most ? most : n;
  n = n < least ? least : n;
  n = n > kMaxSplits ? kMaxSplits : n;
  const int64_t per = exl3h::align_up((size_t)((vocab + n - 1) / n), 8);
  return Split{(int)((vocab + per - 1) / per), (int)per};
}

struct SampleWs {
  size_t best, min_mass, mass, place, group_mass, group_count, order, total;
};

SampleWs sample_ws(int64_t rows, int64_t vocab) {
  const Split sp = split_of(rows, vocab);
  const size_t n = (size_t)rows * sp.splits;
  SampleWs w;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += exl3h::align_up(bytes, 256);
    return here;
  };
  w.best = take(n * 8);
  w.min_mass = take(n * 8);
  w.mass = take(n * kBins * 8);
  w.place = take(n * kBins * 4);
  w.group_mass = take(n * kGroups * 8);
  w.group_count = take(n * kGroups * 4);
  w.order = take(n * sp.per_split * 2);
  w.total = at;
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
  // outputs and workspace apart from the logits and each other
  const struct {
    const void *p;
    size_t bytes;
  } parts[5] = {{logits, (size_t)((rows - 1) * row_stride + vocab) * size}, {u, (size_t)rows * 4},
                {ids, (size_t)rows * 4}, {probs, probs ? (size_t)rows * 4 : 0}, {workspace, w.total}};
  for (int i = 2; i < 5; ++i)
    for (int j = 0; j < i; ++j)
      if (spans_meet(parts[i].p, parts[i].bytes, parts[j].p, parts[j].bytes))
        return fail(EXL3_ERR_INVALID, "exl3_sample: ids, probs or the workspace overlaps another argument");
  SampleArgs a = {};
  a.logits = logits;
  a.rows = rows;
  a.stride = row_stride;
  a.vocab = (int32_t)vocab;
  const Split sp = split_of(rows, vocab);
  a.splits = sp.splits;
  a.per_split = sp.per_split;
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
  a.place = reinterpret_cast<uint32_t *>(ws + w.place);
  a.group_mass = reinterpret_cast<u64 *>(ws + w.group_mass);
  a.group_count = reinterpret_cast<uint32_t *>(ws + w.group_count);
  a.order = reinterpret_cast<uint16_t *>(ws + w.order);
  auto go = [&](auto e) {
    using E = decltype(e);
    const dim3 grid((unsigned)a.splits, (unsigned)rows);
    const hipStream_t st = stream_of(stream);
    k_sample_max<E><<<grid, kThreads, 0, st>>>(a);
    if (cfg->temperatures || cfg->temperature > 0.0f) k_sample_hist<E><<<grid, kThreads, 0, st>>>(a);
    k_sample_pick<E><<<(unsigned)rows, kThreads, 0, st>>>(a);
  };
  if (cfg->dtype == EXL3_ST_F32) go(float{});
  else with_elem16(cfg->dtype, go);
  EXL3_LAUNCHED("k_sample");
  return EXL3_OK;
}

}  // extern "C"
