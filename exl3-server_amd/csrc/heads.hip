// The norm of every query and key head with the position rotation behind it (gfx950).
//
//   y = x * r * w,  r = 1 / sqrt(mean(x^2) + eps) (RMS) or 1 / sqrt(sum(x^2) + eps) (L2)
//   of the first R values of a head, pairs (a, b) = (y[i], y[i + R/2]) or (y[2i], y[2i + 1]):
//   (a cos - b sin, b cos + a sin), angle = position * inv_freq[i]
//
// Statistics, products and the rotation are f32; the result is rounded once. An angle is
// taken in f64 and reduced to turns there: position * inv_freq has up to 55 bits, and at
// position 10^6 an f32 product is off by 0.06 of a radian.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "elem.hpp"
#include "exl3_device.hpp"
#include "exl3_internal.hpp"
#include "exl3_moe.h"

using namespace exl3d;
using namespace exl3e;

namespace {

constexpr int kMaxHeadDim = 1024;
constexpr int64_t kMaxSpan = (int64_t)1 << 48;  // elements that a side's tokens or heads span
constexpr int64_t kMostTokens = 1 << 22;        // of a launch, which holds 2^32 threads in a dimension
constexpr int kMaxFastDim = 512;  // 64 lanes of 8 values
constexpr int kThreads = 256;
constexpr int kEnough = 4096;     // workgroups, 16 a CU: 2048 tokens of 128 heads 33 us, with 2048 workgroups 35, with 16384 36

struct HeadSide {
  const void *x, *w;
  void *y;
  int32_t heads;
  int64_t x_token, x_head, y_token, y_head;
};

struct HeadArgs {
  HeadSide s[2];
  int32_t d, R, interleaved;
  float mean, eps;  // mean: 1 / d, or 1 for the L2 norm
  const int32_t *positions;
  const float *inv_freq;
};

// cos and sin of position * inv_freq.
__device__ __forceinline__ float2 turn(int32_t pos, float inv_freq) {
  const double t = (double)pos * (double)inv_freq * 0.15915494309189533577;  // in turns
  float s, c;
  sincospif((float)(2.0 * (t - rint(t))), &s, &c);
  return make_float2(c, s);
}

__device__ __forceinline__ float scale_of(const HeadArgs &a, float sq) {
  return __builtin_amdgcn_rsqf(fmaf(sq, a.mean, a.eps));
}

// Any head size up to 1024, any strides: a wave per head, values one by one, the normed head
// in LDS for the rotation's partners.
template <typename E>
__global__ __launch_bounds__(64) void k_head_norm_any(HeadArgs a) {
  __shared__ float y[kMaxHeadDim];
  const int lane = threadIdx.x;
  const int64_t tok = blockIdx.x;
  const int h = blockIdx.y;
  const bool second = h >= a.s[0].heads;
  const HeadSide &s = a.s[second ? 1 : 0];
  const int hh = second ? h - a.s[0].heads : h;
  const E *x = reinterpret_cast<const E *>(s.x) + tok * s.x_token + hh * s.x_head;
  const E *w = reinterpret_cast<const E *>(s.w);
  E *out = reinterpret_cast<E *>(s.y) + tok * s.y_token + hh * s.y_head;
  float sq = 0.0f;
  for (int i = lane; i < a.d; i += 64) {
    const float v = to_f32(x[i]);
    y[i] = v;
    sq = fmaf(v, v, sq);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sq += __shfl_xor(sq, o);
  const float r = scale_of(a, sq);
  for (int i = lane; i < a.d; i += 64) y[i] = y[i] * r * (w ? to_f32(w[i]) : 1.0f);
  __syncthreads();
  const int half = a.R / 2;
  for (int i = lane; i < half; i += 64) {
    const float2 cs = turn(a.positions[tok], a.inv_freq[i]);
    const int p = a.interleaved ? 2 * i : i, q = a.interleaved ? 2 * i + 1 : i + half;
    const float u = y[p], v = y[q];
    out[p] = from_f32<E>(u * cs.x - v * cs.y);
    out[q] = from_f32<E>(v * cs.x + u * cs.y);
  }
  for (int i = a.R + lane; i < a.d; i += 64) out[i] = from_f32<E>(y[i]);
}

// Byte distance from the first to past the last value of a side's rows.
size_t span_bytes(const HeadSide &s, bool out, int64_t T, int d) {
  const int64_t t = out ? s.y_token : s.x_token, h = out ? s.y_head : s.x_head;
  return (size_t)((T - 1) * t + (s.heads - 1) * h + d) * 2;
}

// Heads of up to 512 values in groups of 8, at 16-byte addresses: kLanes lanes of 8 values each
// (a power of two; lanes past the head are idle) hold a head in registers, 256 / kLanes heads a
// workgroup at once. A token's angles are computed once for all of a workgroup's heads, while
// the first heads' values are on their way. The partners of a rotation by halves are read
// again (from the first-level cache), which costs less than 8 lane exchanges; a head's lanes are
// of one wave, whose loads are done before its stores, so that works in place as well.
// Bound by HBM for many tokens (2048 of 128 heads of 128: 134 MB in 31 us, 4.3 TB/s), by latency
// for few (one token 2.9 us). kPast: the results go past the caches.
template <typename E, int kLanes, bool kPast>
__global__ __launch_bounds__(kThreads) void k_head_norm(HeadArgs a, int per_group) {
  constexpr int kAtOnce = kThreads / kLanes;
  __shared__ float2 turns[kMaxFastDim / 2];
  const int64_t tok = blockIdx.x;
  const int l = threadIdx.x % kLanes, e = 8 * l, half = a.R / 2, all = a.s[0].heads + a.s[1].heads;
  const int first = blockIdx.y * per_group + threadIdx.x / kLanes, last = min(all, (int)(blockIdx.y + 1) * per_group);
  // this lane's rotation: of pairs inside it, with the half behind or before it, or none
  const bool pairs = a.interleaved && e < a.R, later = !a.interleaved && e >= half && e < a.R;
  const bool halves = !a.interleaved && e < a.R;
  const int other = later ? e - half : e + half;
  auto row = [&](int h, const HeadSide *&s, const E *&x) {
    const bool second = h >= a.s[0].heads;
    s = &a.s[second];
    const int hh = second ? h - a.s[0].heads : h;
    x = reinterpret_cast<const E *>(s->x) + tok * s->x_token + hh * s->x_head;
    return hh;
  };
  float x[8] = {}, p[8] = {};
  auto fetch = [&](int h) {
    const HeadSide *s;
    const E *at;
    row(h, s, at);
    if (e < a.d) load8(at + e, x);
    if (halves) load8(at + other, p);
  };
  if (first < last) fetch(first);
  if (a.R) {
    const int32_t pos = a.positions[tok];
    for (int i = threadIdx.x; i < half; i += kThreads) turns[i] = turn(pos, a.inv_freq[i]);
    __syncthreads();
  }
  for (int h = first; h < last; h += kAtOnce) {
    const HeadSide *s;
    const E *at;
    const int hh = row(h, s, at);
    float sq = 0.0f, y[8], o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = x[i];
      o[i] = p[i];
      sq = fmaf(x[i], x[i], sq);
    }
    if (h + kAtOnce < last) fetch(h + kAtOnce);
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1) sq += __shfl_xor(sq, m);
    const float r = scale_of(a, sq);
    const E *w = reinterpret_cast<const E *>(s->w);
    if (e >= a.d) continue;
    float wv[8];
    if (w) load8(w + e, wv);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] * r * (w ? wv[i] : 1.0f);
    if (pairs) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        if (e + i < a.R) {
          const float2 cs = turns[e / 2 + i / 2];
          const float u = y[i], v = y[i + 1];
          y[i] = u * cs.x - v * cs.y;
          y[i + 1] = v * cs.x + u * cs.y;
        }
      }
    } else if (halves) {
      if (w) load8(w + other, wv);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 cs = turns[(later ? other : e) + i];
        const float v = o[i] * r * (w ? wv[i] : 1.0f);
        y[i] = later ? y[i] * cs.x + v * cs.y : y[i] * cs.x - v * cs.y;
      }
    }
    store8<kPast>(reinterpret_cast<E *>(s->y) + tok * s->y_token + hh * s->y_head + e, y);
  }
}

// Whether a side's rows and weights lie at 16-byte addresses.
bool aligned16(const HeadSide &s) {
  return (reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.y) | reinterpret_cast<uintptr_t>(s.w)) % 16 == 0 &&
         (s.x_token | s.x_head | s.y_token | s.y_head) % 8 == 0;
}

// Whether two sides' rows share a value: exactly where both are token-major with one token
// stride (parts of one packed row), else where their spans meet.
bool rows_meet(const void *pa, int64_t ta, int64_t ha, int na, const void *pb, int64_t tb, int64_t hb, int nb,
               int64_t T, int d) {
  const int64_t wa = (na - 1) * ha + d, wb = (nb - 1) * hb + d;
  const uintptr_t a = reinterpret_cast<uintptr_t>(pa), b = reinterpret_cast<uintptr_t>(pb);
  if (ta != tb || ta < wa || ta < wb || T == 1)
    return spans_meet(a, (size_t)((T - 1) * ta + wa) * 2, b, (size_t)((T - 1) * tb + wb) * 2);
  const int64_t delta = (int64_t)(b - a), s = 2 * ta;
  int64_t q = delta / s, r = delta % s;
  if (r < 0) {
    r += s;
    --q;
  }
  // b's row t begins r bytes behind a's row t + q, and s - r bytes before a's row t + q + 1
  return (r < 2 * wa && std::llabs(q) < T) || (s - r < 2 * wb && std::llabs(q + 1) < T);
}

}  // namespace

using namespace exl3h;

extern "C" exl3_status exl3_head_norm(const exl3_head_norm_config *cfg, const exl3_head_rows *q, const exl3_head_rows *k,
                                      int64_t tokens, const int32_t *positions, const float *inv_freq,
                                      exl3_stream_t stream) {
  if (!cfg || !q) return fail(EXL3_ERR_INVALID, "exl3_head_norm: null argument");
  if (cfg->dtype != EXL3_ST_F16 && cfg->dtype != EXL3_ST_BF16)
    return fail(EXL3_ERR_UNSUPPORTED, "exl3_head_norm: dtype must be f16 or bf16");
  if (cfg->mode != EXL3_NORM_RMS && cfg->mode != EXL3_NORM_L2)
    return fail(EXL3_ERR_INVALID, "exl3_head_norm: unknown mode");
  const int d = cfg->head_dim;
  if (d < 1 || d > kMaxHeadDim) return fail(EXL3_ERR_UNSUPPORTED, "exl3_head_norm: head_dim must be 1..1024");
  if (cfg->rotate_dims < 0 || cfg->rotate_dims > d || cfg->rotate_dims % 2)
    return fail(EXL3_ERR_INVALID, "exl3_head_norm: rotate_dims must be even and at most head_dim");
  if (!(cfg->eps >= 0.0f)) return fail(EXL3_ERR_INVALID, "exl3_head_norm: eps must not be negative");
  if (tokens < 0 || tokens > ((int64_t)1 << 31) - 1) return fail(EXL3_ERR_INVALID, "exl3_head_norm: bad token count");
  const exl3_head_rows *sides[2] = {q, k};
  HeadArgs a = {};
  a.R = cfg->rotate_dims;
  int heads = 0;
  for (int i = 0; i < (k ? 2 : 1); ++i) {
    const exl3_head_rows &s = *sides[i];
    // head counts of a launch's second dimension
    if (s.heads < 1 || s.heads > 32767) return fail(EXL3_ERR_INVALID, "exl3_head_norm: heads must be 1..32767");
    for (int64_t v : {s.x_token, s.x_head, s.y_token, s.y_head})
      if (v < 0 || v > kMaxSpan / 32768) return fail(EXL3_ERR_INVALID, "exl3_head_norm: bad stride");
    if (tokens && (s.x_token > kMaxSpan / tokens || s.y_token > kMaxSpan / tokens))
      return fail(EXL3_ERR_INVALID, "exl3_head_norm: bad stride");
    const bool token_major = (s.heads == 1 || s.y_head >= d) && (tokens <= 1 || s.y_token >= (s.heads - 1) * s.y_head + d);
    const bool head_major = (tokens <= 1 || s.y_token >= d) && (s.heads == 1 || s.y_head >= (tokens - 1) * s.y_token + d);
    if (!token_major && !head_major) return fail(EXL3_ERR_INVALID, "exl3_head_norm: output rows overlap each other");
    a.s[i] = HeadSide{s.x, s.w, s.y, s.heads, s.x_token, s.x_head, s.y_token, s.y_head};
    heads += s.heads;
  }
  if (tokens == 0) return EXL3_OK;
  for (int i = 0; i < (k ? 2 : 1); ++i) {
    const HeadSide &s = a.s[i];
    if (!s.x || !s.y) return fail(EXL3_ERR_INVALID, "exl3_head_norm: null rows");
    if ((reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.y) | reinterpret_cast<uintptr_t>(s.w)) % 2)
      return fail(EXL3_ERR_INVALID, "exl3_head_norm: rows and weights must be 2-byte aligned");
    for (int j = 0; j < (k ? 2 : 1); ++j) {
      const HeadSide &o = a.s[j];
      const bool in_place = i == j && s.x == s.y && (tokens == 1 || s.x_token == s.y_token) && (s.heads == 1 || s.x_head == s.y_head);
      if (!in_place && rows_meet(s.y, s.y_token, s.y_head, s.heads, o.x, o.x_token, o.x_head, o.heads, tokens, d))
        return fail(EXL3_ERR_INVALID, "exl3_head_norm: an output overlaps an input (in place: the same rows)");
      if (o.w && spans_meet(reinterpret_cast<uintptr_t>(s.y), span_bytes(s, true, tokens, d),
                            reinterpret_cast<uintptr_t>(o.w), (size_t)d * 2))
        return fail(EXL3_ERR_INVALID, "exl3_head_norm: an output overlaps a weight");
    }
  }
  if (k && rows_meet(a.s[0].y, a.s[0].y_token, a.s[0].y_head, a.s[0].heads, a.s[1].y, a.s[1].y_token, a.s[1].y_head,
                     a.s[1].heads, tokens, d))
    return fail(EXL3_ERR_INVALID, "exl3_head_norm: the outputs overlap each other");
  if (cfg->rotate_dims) {
    if (!positions || !inv_freq) return fail(EXL3_ERR_INVALID, "exl3_head_norm: the rotation needs positions and inv_freq");
    if ((reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(inv_freq)) % 4)
      return fail(EXL3_ERR_INVALID, "exl3_head_norm: positions and inv_freq must be 4-byte aligned");
  }
  for (int i = 0; i < (k ? 2 : 1) && a.R; ++i) {
    const uintptr_t y = reinterpret_cast<uintptr_t>(a.s[i].y);
    const size_t bytes = span_bytes(a.s[i], true, tokens, d);
    if (spans_meet(y, bytes, reinterpret_cast<uintptr_t>(positions), (size_t)tokens * 4) ||
        spans_meet(y, bytes, reinterpret_cast<uintptr_t>(inv_freq), (size_t)a.R * 2))
      return fail(EXL3_ERR_INVALID, "exl3_head_norm: an output overlaps positions or inv_freq");
  }
  a.d = d;
  a.interleaved = cfg->interleaved != 0;
  a.mean = cfg->mode == EXL3_NORM_L2 ? 1.0f : 1.0f / (float)d;
  a.eps = cfg->eps;
  a.inv_freq = inv_freq;
  // Results that the L2s (8 of 4 MB) would not hold: past them, 2048 tokens of 128 heads of 128
  // take 33 us and not 42 (a copy of as many bytes: 28).
  const bool past = tokens * heads * d * 2 > (32 << 20);
  const HeadSide whole[2] = {a.s[0], a.s[1]};
  with_elem16(cfg->dtype, [&](auto e) {
    using E = decltype(e);
    const hipStream_t st = stream_of(stream);
    // (halves that end inside a lane's 8 values take the general kernel)
    const bool halves_fit = a.interleaved || a.R % 16 == 0;
    const bool fast = d % 8 == 0 && d <= kMaxFastDim && halves_fit && aligned16(a.s[0]) && (!k || aligned16(a.s[1]));
    for (int64_t t0 = 0; t0 < tokens; t0 += kMostTokens) {
      const int64_t n = tokens - t0 < kMostTokens ? tokens - t0 : kMostTokens;
      a.positions = a.R ? positions + t0 : nullptr;
      for (int i = 0; i < (k ? 2 : 1); ++i) {
        a.s[i].x = reinterpret_cast<const E *>(whole[i].x) + t0 * whole[i].x_token;
        a.s[i].y = reinterpret_cast<E *>(whole[i].y) + t0 * whole[i].y_token;
      }
      if (!fast) {
        k_head_norm_any<E><<<dim3((unsigned)n, (unsigned)heads), 64, 0, st>>>(a);
        continue;
      }
      auto go = [&](auto lanes) {
        constexpr int kLanes = decltype(lanes)::value, kAtOnce = kThreads / kLanes;
        // heads of a workgroup: as many as leave enough workgroups
        const int64_t passes = (heads + kAtOnce - 1) / kAtOnce;
        int64_t groups = (kEnough + n - 1) / n;
        groups = groups < passes ? groups : passes;
        const int per_group = (int)((passes + groups - 1) / groups) * kAtOnce;
        const dim3 grid((unsigned)n, (unsigned)((heads + per_group - 1) / per_group));
        if (past) k_head_norm<E, kLanes, true><<<grid, kThreads, 0, st>>>(a, per_group);
        else k_head_norm<E, kLanes, false><<<grid, kThreads, 0, st>>>(a, per_group);
      };
      if (d <= 64) go(std::integral_constant<int, 8>{});
      else if (d <= 128) go(std::integral_constant<int, 16>{});
      else if (d <= 256) go(std::integral_constant<int, 32>{});
      else go(std::integral_constant<int, 64>{});
    }
  });
  EXL3_LAUNCHED("k_head_norm");
  return EXL3_OK;
}
