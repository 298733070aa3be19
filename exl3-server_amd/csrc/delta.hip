// The gated delta rule over a batch of sequences of any lengths (gfx950).
//
// A head's state S (dk, dv) is f32. For each token, with a = exp(g) (one decay for the head,
// or one per key channel):
//   S <- diag(a) S;  u = beta (v - S^T k);  S <- S + k u^T;  out = scale S^T q
//
//  k_delta_step   token by token: the state in registers from its slot to its slot.
//  k_delta_chunk, k_delta_scan   chunks of C = 32 tokens. With the chunk's first state S0, the
//    running products P_i = a_1 .. a_i and U the rows u of the rule:
//      A_ij = k_i . (P_i / P_j) k_j (j < i),  B_ij = q_i . (P_i / P_j) k_j (j <= i)
//      U = T diag(beta) (V - (P K) S0),  T = (I + diag(beta) A)^-1
//      out = scale ((P Q) S0 + B U),  S <- diag(P_C) S0 + (P_C / P K)^T U
//    k_delta_chunk computes T and B of every chunk and head side by side; k_delta_scan goes
//    through a sequence's chunks with its state in registers.
//
// A ratio P_i / P_j is never a quotient nor a difference of sums of g: it is the product
// of the decays between, which stays exact where a decay is 0 (g = -inf) or tiny.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "elem.hpp"
#include "exl3_device.hpp"
#include "exl3_internal.hpp"
#include "exl3_moe.h"

using namespace exl3d;
using namespace exl3e;

namespace {

constexpr int kCols = 16;  // state columns of a wave

struct ChunkMats;

struct DeltaArgs {
  const void *q, *k, *v;
  const float *g, *beta;
  void *out;
  int64_t q_token, k_token, v_token, g_token, beta_token, out_token;
  int32_t tokens, n_seq, heads_qk, heads_v, dv;
  float scale;
  const int32_t *starts;  // NULL: sequences of tokens / n_seq
  float *state;
  int64_t n_slots;
  const int32_t *src, *dst;
  ChunkMats *chunks;  // (chunk ids, heads_v)
  int32_t chunked;    // sequences of at least so many tokens go in chunks, the others in steps
  int32_t scanned;    // at most so many sequences go in chunks
  bool words;         // q's and k's rows begin at 4-byte addresses
};

struct Seq {
  int first, last;  // tokens [first, last)
};

// A sequence's tokens; whatever `starts` holds they lie in the call's.
__device__ __forceinline__ Seq seq_of(const DeltaArgs &a, int i) {
  if (!a.starts) {
    const int n = a.tokens / a.n_seq;
    return Seq{i * n, i * n + n};
  }
  const int first = min(max(a.starts[i], 0), a.tokens);
  return Seq{first, min(max(a.starts[i + 1], first), a.tokens)};
}

__device__ __forceinline__ int64_t slot_of(const int32_t *slots, int i, int64_t n_slots) {
  const int64_t s = slots ? slots[i] : i;
  return s >= 0 && s < n_slots ? s : -1;
}

// Whether sequence i may write its slot: one that another sequence reads or writes in the
// same call keeps its old state. Called by every thread of a workgroup.
__device__ __forceinline__ bool sole_writer(const DeltaArgs &a, int i, int64_t slot) {
  if (slot < 0) return false;
  bool met = false;
  for (int j = threadIdx.x; j < a.n_seq; j += blockDim.x)
    if (j != i) met |= slot_of(a.src, j, a.n_slots) == slot || slot_of(a.dst, j, a.n_slots) == slot;
  return !__syncthreads_or(met);
}

// The j-th sequence that goes in chunks, or -1. Called by every thread of a workgroup of 512.
__device__ __forceinline__ int nth_chunked(const DeltaArgs &a, int j) {
  __shared__ int found, count[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) found = -1;
  for (int first = 0; first < a.n_seq; first += 512) {
    const int i = first + tid;
    const Seq s = seq_of(a, min(i, a.n_seq - 1));
    const bool own = i < a.n_seq && s.last - s.first >= a.chunked;
    const uint64_t lanes = __ballot(own);
    if (lane == 0) count[wave] = __popcll(lanes);
    __syncthreads();
    int before = __popcll(lanes & (((uint64_t)1 << lane) - 1)), all = 0;
    for (int w = 0; w < 8; ++w) {
      if (w < wave) before += count[w];
      all += count[w];
    }
    if (own && before == j) found = i;
    j -= all;
    __syncthreads();
  }
  return found;
}

// x + the partner's x, of lane ^ 16 and of lane ^ 32: an exchange holds both, in either order.
__device__ __forceinline__ float add_16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(bitcast<uint32_t>(x), bitcast<uint32_t>(x), false, false);
  return bitcast<float>(r[0]) + bitcast<float>(r[1]);
}
__device__ __forceinline__ float add_32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(bitcast<uint32_t>(x), bitcast<uint32_t>(x), false, false);
  return bitcast<float>(r[0]) + bitcast<float>(r[1]);
}

// Sum over the 16 lanes of a wave that hold the same columns (lane / 4), the same bits in all:
// rows of 16 lanes turned by 8 (lane ^ 8), by 4 (as lane ^ 4 then), and the rows. No LDS.
__device__ __forceinline__ f32x4 sum_rows(f32x4 v) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float x = v[c];
    x += bitcast<float>(__builtin_amdgcn_mov_dpp(bitcast<int>(x), 0x128, 0xF, 0xF, false));
    x += bitcast<float>(__builtin_amdgcn_mov_dpp(bitcast<int>(x), 0x124, 0xF, 0xF, false));
    v[c] = add_32(add_16(x));
  }
  return v;
}

// A wave holds kCols columns of the state: lane l the columns 4 (l % 4).. and the DK / 16
// rows from (l / 4) DK / 16, so that a token needs two sums over 16 lanes and no barrier.
// Bound by the states' traffic for many sequences (64 of 64 heads of 128 x 128: 537 MB read and
// written in 108 us a call, 5.0 TB/s, a large copy's rate), by latencies for few (one
// sequence 5.1 us; 8 of 16 heads with 4 tokens each 9.1-10).
template <typename E, int DK, bool kChannel>
__global__ __launch_bounds__(256) void k_delta_step(DeltaArgs a) {
  constexpr int R = DK / 16;
  const int lane = threadIdx.x & 63, seq = blockIdx.z, h = blockIdx.y, hk = h / (a.heads_v / a.heads_qk);
  const Seq s = seq_of(a, seq);
  if (s.last - s.first >= a.chunked) return;
  const int64_t from = slot_of(a.src, seq, a.n_slots), to = slot_of(a.dst, seq, a.n_slots);
  const bool write = sole_writer(a, seq, to);
  const int block = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (block * kCols >= a.dv) return;
  const int row = lane / 4 * R, col = block * kCols + lane % 4 * 4;
  const size_t head = (size_t)DK * a.dv, at = h * head + (size_t)row * a.dv + col;
  f32x4 S[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    S[r] = from < 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f}
                    : *reinterpret_cast<const f32x4 *>(a.state + from * a.heads_v * head + at + (size_t)r * a.dv);
  const E *q = reinterpret_cast<const E *>(a.q) + (int64_t)hk * DK + row;
  const E *k = reinterpret_cast<const E *>(a.k) + (int64_t)hk * DK + row;
  const E *v = reinterpret_cast<const E *>(a.v) + (int64_t)h * a.dv + col;
  E *out = reinterpret_cast<E *>(a.out) + (int64_t)h * a.dv + col;
  const float *g = a.g + (kChannel ? (int64_t)h * DK + row : h);
  // a token's rows, the next one's loaded while this one's are computed on
  typedef E ER __attribute__((ext_vector_type(R), aligned(2)));
  typedef E E4 __attribute__((ext_vector_type(4), aligned(2)));
  typedef float GR __attribute__((ext_vector_type(kChannel ? R : 1), aligned(4)));
  struct Token {
    ER k, q;
    GR g;
    E4 v;
    float beta;
  };
  auto load = [&](int64_t t) {
    return Token{*reinterpret_cast<const ER *>(k + t * a.k_token), *reinterpret_cast<const ER *>(q + t * a.q_token),
                 *reinterpret_cast<const GR *>(g + t * a.g_token), *reinterpret_cast<const E4 *>(v + t * a.v_token),
                 a.beta[t * a.beta_token + h]};
  };
  Token next;
  if (s.first < s.last) next = load(s.first);
  for (int64_t t = s.first; t < s.last; ++t) {
    const Token now = next;
    next = load(t + 1 < s.last ? t + 1 : t);
    float kk[R], qq[R], decay[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      kk[r] = to_f32((E)now.k[r]);
      qq[r] = to_f32((E)now.q[r]);
      decay[r] = now.g[kChannel ? r : 0];
    }
    const float beta = now.beta;
    f32x4 vv;
#pragma unroll
    for (int c = 0; c < 4; ++c) vv[c] = to_f32((E)now.v[c]);
    f32x4 dot = {0.0f, 0.0f, 0.0f, 0.0f}, o = dot;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float d = expf(decay[r]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        S[r][c] *= d;
        dot[c] = fmaf(kk[r], S[r][c], dot[c]);
      }
    }
    dot = sum_rows(dot);
    f32x4 u;
#pragma unroll
    for (int c = 0; c < 4; ++c) u[c] = beta * (vv[c] - dot[c]);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        S[r][c] = fmaf(kk[r], u[c], S[r][c]);
        o[c] = fmaf(qq[r], S[r][c], o[c]);
      }
    o = sum_rows(o);
    if (lane < 4) {
#pragma unroll
      for (int c = 0; c < 4; ++c) out[t * a.out_token + c] = from_f32<E>(a.scale * o[c]);
    }
  }
  if (write)
#pragma unroll
    for (int r = 0; r < R; ++r)
      *reinterpret_cast<f32x4 *>(a.state + to * a.heads_v * head + at + (size_t)r * a.dv) = S[r];
}

// --- chunks ---------------------------------------------------------------------------

constexpr int kC = 32;               // tokens of a chunk
constexpr int kPad = 4;              // words behind an f32 LDS row: 16-byte reads of 16 rows meet no bank twice

// The scan multiplies f16 pairs: x = hi + lo, hi = f16(x), lo = f16(x - hi), 22 bits of x, and
// three of the four products (lo lo is under 2^-22 of the result). Keys, queries, T and B
// go in times 2^6, which leaves an error of at most 2^-31 where lo is a subnormal; state columns
// and the rows between by a power of two that brings the column's largest value to 2^13.
// A chunk whose values lie outside is done token by token in f32: |k|, |q|, |T|, |B| of 2^9 or
// more, decays over 1, a key whose largest value is under 2^-8 (2^-31 is 2^-23 of that) or a
// query's under 2^-16 (2^-15, of a result with 11 bits), unless all its values are 0.
constexpr float kScale = 64.0f, kLimit = 512.0f, kLeastKey = 0x1p-8f, kLeastQuery = 0x1p-16f;
// Of one chunk and head, in the workspace: T and B as hi and lo, the columns in operand order,
// and two marks of a chunk that the scan may multiply.
struct ChunkMats {
  f16 mat[4][kC][kC];  // T hi, T lo, B hi, B lo
  float beta[kC];
  int32_t fine[4];     // [0], [1] used
};
static_assert(sizeof(ChunkMats) % 16 == 0, "16-byte loads");
// Where the instruction's k index i (of 32) is in operand order: lane group g takes the indices
// 4 g .. 4 g + 3 and 16 + 4 g .., which are the rows that a result's lane group holds.
__device__ __forceinline__ constexpr int in_order(int i) {
  return (i & 12) * 2 + (i & 3) + (i >> 4 & 1) * 4 + (i & ~31);
}

typedef f16 f16x8 __attribute__((ext_vector_type(8)));
struct Pair {
  f16x8 hi, lo;
};

// Chunk c of sequence i has id first / C + i + c: distinct over the call, under tokens / C + n_seq.
__device__ __forceinline__ int first_chunk(const Seq &s, int i) { return s.first / kC + i; }
__device__ __forceinline__ int chunks_of(const Seq &s) { return (s.last - s.first + kC - 1) / kC; }

// exp(g). (The product's rounding costs |g| 2^-24 of a factor exp(g): at most 2^-25.)
__device__ __forceinline__ float decay_of(float g) { return __builtin_amdgcn_exp2f(g * 1.44269504f); }

// A uniform value that the compiler cannot see to be one.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The first of a chunk's rows of `stride` elements of E, at head offset `at` (uniform).
template <typename E>
__device__ __forceinline__ const char *chunk_rows(const void *p, int64_t stride, int t0, int64_t at) {
  return reinterpret_cast<const char *>(p) + (t0 * stride + at) * (int64_t)sizeof(E);
}

// The DK / 64 channels of 8 tokens that a lane holds, as they lie in memory: loaded a chunk
// ahead and converted when they are taken, so that no load is waited for one by one. Tokens
// behind the chunk's n read its last row's values, to be cleared.
template <typename E, int DK, bool kChannel>
struct RawSlice {
  static constexpr int N = DK / 64, G = kChannel ? N : 1;
  typedef E EN __attribute__((ext_vector_type(N), aligned(2)));
  typedef float GN __attribute__((ext_vector_type(G), aligned(4)));
  EN k[8], q[8];
  GN g[8];

  // tokens from n on: zeros with decay 1
  __device__ __forceinline__ void clear(int n, int tok) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (tok + i >= n) {
#pragma unroll
        for (int c = 0; c < N; ++c) k[i][c] = q[i][c] = from_f32<E>(0.0f);
#pragma unroll
        for (int c = 0; c < G; ++c) g[i][c] = 0.0f;
      }
  }
  // chunk tokens tok .., channels ch ..
  __device__ __forceinline__ void load(const DeltaArgs &a, int t0, int n, int h, int hk, int tok, int ch) {
    const char *kb = chunk_rows<E>(a.k, a.k_token, t0, (int64_t)hk * DK);
    const char *qb = chunk_rows<E>(a.q, a.q_token, t0, (int64_t)hk * DK);
    const char *gb = chunk_rows<float>(a.g, a.g_token, t0, kChannel ? (int64_t)h * DK : h);
    const uint32_t ks = (uint32_t)a.k_token * 2, qs = (uint32_t)a.q_token * 2, gs = (uint32_t)a.g_token * 4;
    const uint32_t c2 = ch * 2, c4 = kChannel ? ch * 4 : 0;
    if (a.words) {
      // rows at 4-byte addresses: what lies behind the last one reads as zeros (a decay of 1)
      auto rows = [&](const char *p, uint32_t stride, uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc((void *)p, (short)0, (int)(uniform(min(n, kC) - 1) * stride + bytes), 0x00020000);
      };
      const __amdgpu_buffer_rsrc_t kr = rows(kb, ks, DK * 2), qr = rows(qb, qs, DK * 2), gr = rows(gb, gs, kChannel ? DK * 4 : 4);
      const int ko = tok * ks + c2, qo = tok * qs + c2, go = tok * gs + c4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (N == 2) {
          k[i] = bitcast<EN>((uint32_t)__builtin_amdgcn_raw_buffer_load_b32(kr, ko + i * ks, 0, 0));
          q[i] = bitcast<EN>((uint32_t)__builtin_amdgcn_raw_buffer_load_b32(qr, qo + i * qs, 0, 0));
        } else {
          k[i] = bitcast<EN>((uint16_t)__builtin_amdgcn_raw_buffer_load_b16(kr, ko + i * ks, 0, 0));
          q[i] = bitcast<EN>((uint16_t)__builtin_amdgcn_raw_buffer_load_b16(qr, qo + i * qs, 0, 0));
        }
        if constexpr (G == 2) g[i] = bitcast<GN>(__builtin_amdgcn_raw_buffer_load_b64(gr, go + i * gs, 0, 0));
        else g[i] = bitcast<GN>(__builtin_amdgcn_raw_buffer_load_b32(gr, go + i * gs, 0, 0));
      }
    } else if (n >= kC) {
      const uint32_t ko = tok * ks + c2, qo = tok * qs + c2, go = tok * gs + c4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        k[i] = *reinterpret_cast<const EN *>(kb + (ko + i * ks));
        q[i] = *reinterpret_cast<const EN *>(qb + (qo + i * qs));
        g[i] = *reinterpret_cast<const GN *>(gb + (go + i * gs));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t t = min(tok + i, n - 1);
        k[i] = *reinterpret_cast<const EN *>(kb + (t * ks + c2));
        q[i] = *reinterpret_cast<const EN *>(qb + (t * qs + c2));
        g[i] = *reinterpret_cast<const GN *>(gb + (t * gs + c4));
      }
    }
  }
};

// The same in f32, and the decays' running products in blocks of `h` tokens: up to and with
// token i (P), and behind it (X).
template <typename E, int DK, bool kChannel>
struct Slice {
  static constexpr int N = DK / 64;
  float k[8][N], q[8][N], P[8][N], X[8][N];

  // blocks of one token
  __device__ __forceinline__ void convert(const RawSlice<E, DK, kChannel> &x) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < N; ++c) {
        k[i][c] = to_f32((E)x.k[i][c]);
        q[i][c] = to_f32((E)x.q[i][c]);
        P[i][c] = kChannel || c == 0 ? decay_of(x.g[i][c % RawSlice<E, DK, kChannel>::G]) : P[i][0];
        X[i][c] = 1.0f;
      }
  }
  // Whether the scan may multiply these values, by their bits: magnitudes order as integers,
  // infinities and NaN above all others. Called by whole waves that hold whole tokens.
  __device__ __forceinline__ bool fine(const RawSlice<E, DK, kChannel> &x) const {
    typedef uint16_t U __attribute__((ext_vector_type(N)));
    typedef uint16_t U2 __attribute__((ext_vector_type(2)));
    U2 most[8];  // of token i's key and query
    uint32_t decay = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const U k = bitcast<U>(x.k[i]) & (uint16_t)0x7fff, q = bitcast<U>(x.q[i]) & (uint16_t)0x7fff;
      most[i] = U2{k[0], q[0]};
      if constexpr (N == 2) most[i] = __builtin_elementwise_max(most[i], U2{k[1], q[1]});
#pragma unroll
      for (int n = 0; n < N; ++n) decay = max(decay, bitcast<uint32_t>(P[i][n]));
    }
    // over the wave: halves and rows exchanged with half of the tokens each, then within 16 lanes
    auto larger = [](uint32_t a, uint32_t b) { return __builtin_elementwise_max(bitcast<U2>(a), bitcast<U2>(b)); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto r = __builtin_amdgcn_permlane32_swap(bitcast<uint32_t>(most[i]), bitcast<uint32_t>(most[i + 4]), false, false);
      most[i] = larger(r[0], r[1]);
    }
    bool ok = decay <= 0x3f800000u;  // 1.0f
    const uint16_t limit = bitcast<uint16_t>(from_f32<E>(kLimit));
    const uint16_t key = bitcast<uint16_t>(from_f32<E>(kLeastKey)), query = bitcast<uint16_t>(from_f32<E>(kLeastQuery));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const auto r = __builtin_amdgcn_permlane16_swap(bitcast<uint32_t>(most[i]), bitcast<uint32_t>(most[i + 2]), false, false);
      uint32_t m = bitcast<uint32_t>(larger(r[0], r[1]));
      m = bitcast<uint32_t>(larger(m, __builtin_amdgcn_mov_dpp(m, 0xB1, 0xF, 0xF, false)));
      m = bitcast<uint32_t>(larger(m, __builtin_amdgcn_mov_dpp(m, 0x4E, 0xF, 0xF, false)));
      m = bitcast<uint32_t>(larger(m, __builtin_amdgcn_mov_dpp(m, 0x141, 0xF, 0xF, false)));
      m = bitcast<uint32_t>(larger(m, __builtin_amdgcn_mov_dpp(m, 0x140, 0xF, 0xF, false)));
      const U2 of = bitcast<U2>(m);
      ok = ok && of[0] < limit && of[1] < limit && (of[0] == 0 || of[0] >= key) && (of[1] == 0 || of[1] >= query);
    }
    return ok;
  }
  // from blocks of h to blocks of 2 h tokens (h = 1, 2, 4)
  __device__ __forceinline__ void grow(int h) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int b = i & ~(2 * h - 1);
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (!(i & h)) X[i][n] *= P[b + 2 * h - 1][n];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int b = i & ~(2 * h - 1);
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (i & h) P[i][n] *= P[b + h - 1][n];
    }
  }
};

template <int N>
__device__ __forceinline__ void put(float *p, const float (&v)[N]) {
  if constexpr (N == 2) *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
  else *p = v[0];
}
__device__ __forceinline__ f32x4 mfma4(const f32x4 &a, const f32x4 &b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// A barrier that orders LDS alone: __syncthreads() would also wait for every global load and
// store in flight, which here are the next chunk's.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Where value `col` of an LDS row of left operands lies: the rows' 16-byte pieces are turned
// among themselves so that the 16-byte reads of 16 rows (and the reads of the lane groups beside
// them) meet no bank twice, without padding. Rows of DK channels, and of 32 tokens.
template <int DK>
__device__ __forceinline__ constexpr int channel_at(int row, int col) {
  return col ^ (DK == 128 ? row & 15 : row >> 1 & 7) * 8;
}
__device__ __forceinline__ constexpr int token_at(int row, int col) { return col ^ (-(row >> 2) & 3) * 8; }

// One chunk's left operands in LDS, rows in operand order, and the decay over the chunk.
template <typename E, int DK, int kWaves>
struct alignas(16) Stage {
  static constexpr int kCol = kWaves * kCols + 8;
  f16 pk[2][kC][DK], pq[2][kC][DK];  // P K, P Q: hi, lo (channel_at)
  f16 pe[2][DK][kC];                 // (P_C / P K)^T (token_at)
  f16 mat[4][kC][kC];                // T hi, T lo, B hi, B lo (token_at)
  E v[kC][kCol];
  float decay[DK];
  float beta[kC];
  uint32_t v_bad[4];  // by the wave that carried them: the column blocks in which a value is infinite or NaN
  int fine;
};

// A power of two that brings the largest of a column's values (lanes l, l ^ 16, l ^ 32, ..) to
// [2^13, 2^14), and its inverse. 0, denormals and what is not finite take the nearest that exists.
struct ColumnScale {
  float to, back;
  __device__ __forceinline__ explicit ColumnScale(float most) {
    // the two exchanges hold each lane's own value and its partner's, in either order
    const auto r16 = __builtin_amdgcn_permlane16_swap(bitcast<uint32_t>(most), bitcast<uint32_t>(most), false, false);
    most = fmaxf(bitcast<float>(r16[0]), bitcast<float>(r16[1]));
    const auto r32 = __builtin_amdgcn_permlane32_swap(bitcast<uint32_t>(most), bitcast<uint32_t>(most), false, false);
    most = fmaxf(bitcast<float>(r32[0]), bitcast<float>(r32[1]));
    const uint32_t e = max(bitcast<uint32_t>(most) >> 23, 14u);
    to = bitcast<float>((267u - e) << 23);
    back = bitcast<float>((e - 13u) << 23);
  }
};

__device__ __forceinline__ float most_of(const f32x4 &v, float m) {
#pragma unroll
  for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(v[r]));
  return m;
}

// x s and y s as f16 pairs: hi rounded once, lo the rest of it. hi passes through a register
// that the compiler may not compute twice: a product rounded to f32 first in one place and
// not in the other would leave a lo that fits neither.
__device__ __forceinline__ void split2(float x, float xs, float y, float ys, f16x2 &hi, f16x2 &lo) {
  uint32_t h = bitcast<uint32_t>(f16x2{(f16)(x * xs), (f16)(y * ys)});
  asm("" : "+v"(h));
  hi = bitcast<f16x2>(h);
  lo = f16x2{(f16)fmaf(x, xs, -(float)hi[0]), (f16)fmaf(y, ys, -(float)hi[1])};
}

// Two tiles' results as a right operand (k index in operand order).
__device__ __forceinline__ Pair split(const f32x4 &a, const f32x4 &b, float scale) {
  f16x2 h[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; r += 2) {
    split2(a[r], scale, a[r + 1], scale, h[r / 2], l[r / 2]);
    split2(b[r], scale, b[r + 1], scale, h[2 + r / 2], l[2 + r / 2]);
  }
  Pair p;
#pragma unroll
  for (int r = 0; r < 8; ++r) p.hi[r] = h[r / 2][r % 2], p.lo[r] = l[r / 2][r % 2];
  return p;
}

// c[i] += sum over u of left[u][i] right[u] (lo lo left out), the results' chains in turn.
template <int U, int R>
__device__ __forceinline__ void product(const Pair (&left)[U][R], const Pair (&right)[U], f32x4 (&c)[R]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int i = 0; i < R; ++i) c[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(left[u][i].lo, right[u].hi, c[i], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < R; ++i) c[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(left[u][i].hi, right[u].lo, c[i], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < R; ++i) c[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(left[u][i].hi, right[u].hi, c[i], 0, 0, 0);
  }
}

// N adjacent values v s as f16 pairs.
template <int N>
__device__ __forceinline__ void put_split(f16 *hi, f16 *lo, const float (&v)[N], const float (&sc)[N]) {
  f16x2 h[(N + 1) / 2], l[(N + 1) / 2];
#pragma unroll
  for (int n = 0; n < N; n += 2) split2(v[n], sc[n], v[n + 1 < N ? n + 1 : n], sc[n + 1 < N ? n + 1 : n], h[n / 2], l[n / 2]);
  if constexpr (N == 1) *hi = h[0][0], *lo = l[0][0];
  else {
    typedef uint32_t words __attribute__((ext_vector_type(N / 2)));
    words wh, wl;
    if constexpr (N == 2) wh = bitcast<uint32_t>(h[0]), wl = bitcast<uint32_t>(l[0]);
    else {
#pragma unroll
      for (int n = 0; n < N / 2; ++n) wh[n] = bitcast<uint32_t>(h[n]), wl[n] = bitcast<uint32_t>(l[n]);
    }
    *reinterpret_cast<words *>(hi) = wh;
    *reinterpret_cast<words *>(lo) = wl;
  }
}

// Sums over the wave of 8 values a lane: lane 16 r holds those of value r / 2 * 4 + r % 2 * 2 + i in
// v[i], i = 0, 1. Halves and rows are exchanged with half of the values each, so that
// each step halves what is left.
__device__ __forceinline__ void wave_sums8(float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto r = __builtin_amdgcn_permlane32_swap(bitcast<uint32_t>(v[i]), bitcast<uint32_t>(v[i + 4]), false, false);
    v[i] = bitcast<float>(r[0]) + bitcast<float>(r[1]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto r = __builtin_amdgcn_permlane16_swap(bitcast<uint32_t>(v[i]), bitcast<uint32_t>(v[i + 2]), false, false);
    v[i] = bitcast<float>(r[0]) + bitcast<float>(r[1]);
    // lanes ^ 1, ^ 2, and the mirrors of 8 and of 16 lanes
    v[i] += bitcast<float>(__builtin_amdgcn_mov_dpp(bitcast<int>(v[i]), 0xB1, 0xF, 0xF, false));
    v[i] += bitcast<float>(__builtin_amdgcn_mov_dpp(bitcast<int>(v[i]), 0x4E, 0xF, 0xF, false));
    v[i] += bitcast<float>(__builtin_amdgcn_mov_dpp(bitcast<int>(v[i]), 0x141, 0xF, 0xF, false));
    v[i] += bitcast<float>(__builtin_amdgcn_mov_dpp(bitcast<int>(v[i]), 0x140, 0xF, 0xF, false));
  }
}

// T and B of one chunk and value head. For each h = 1, 2, 4, 8, 16 the pairs (i, j) whose
// highest differing bit is h: i in the later half of a block of 2 h tokens, j in the earlier
// one, so P_i / P_j = (product from the halves' border to i) (product from j to the border),
// both at most 1 for decays that are. The 16 rows with bit h and the 16 without it are one
// tile of the matrix instruction, of which the pairs of a common block are taken. Waves 0
// and 1 multiply A's and B's tiles of h = 1, 4, 16, waves 2 and 3 those of 2 and 8.
// Bound by latencies (its loads, and five levels with a barrier each) at four workgroups a CU:
// 2048 tokens of 64 heads 63-68 us, where its 1.84e7 vector instructions alone would take
// about 30. At five workgroups a CU, with the registers that leaves, 98 against 64 us.
template <typename E, int DK, bool kChannel>
__global__ __launch_bounds__(256, 4) void k_delta_chunk(DeltaArgs a) {
  constexpr int N = DK / 64;
  struct Operands {
    f16 left_k[2][16][DK], left_q[2][16][DK], right[2][16][DK];  // hi, lo, times 2^6 (channel_at)
  };
  struct Results {
    float A[kC][kC + kPad], B[kC][kC + kPad];
    float m00[16][16 + kPad], m11[16][16 + kPad];  // columns
    f16 mat[4][kC][kC];                            // as ChunkMats
    int fine[2];
  };
  union Lds {
    Operands in;
    Results out;
  };
  __shared__ Lds lds;
  __shared__ float total[4][DK];
  __shared__ float beta[kC], diag[kC];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, id = blockIdx.x, h = blockIdx.y;
  int seq = 0;
  if (a.n_seq > 1) {
    __shared__ int of;
    if (tid == 0) of = a.n_seq;
    __syncthreads();
    for (int i = tid; i < a.n_seq; i += 256) {
      const Seq s = seq_of(a, i);
      const int c = id - first_chunk(s, i);
      if (c >= 0 && c < chunks_of(s)) atomicMin(&of, i);
    }
    __syncthreads();
    seq = of;
    if (seq == a.n_seq) return;
  }
  const Seq s = seq_of(a, seq);
  const int chunk = id - first_chunk(s, seq);
  if (chunk < 0 || chunk >= chunks_of(s) || s.last - s.first < a.chunked) return;
  const int t0 = uniform(s.first + chunk * kC), n = uniform(s.last) - t0;
  RawSlice<E, DK, kChannel> raw;
  raw.load(a, t0, n, h, h / (a.heads_v / a.heads_qk), 8 * wave, lane * N);
  float b = 0.0f;
  if (tid < kC) {
    b = tid < n ? a.beta[(int64_t)(t0 + tid) * a.beta_token + h] : 0.0f;
    beta[tid] = b;
  }
  if (n < kC) raw.clear(n, 8 * wave);
  Slice<E, DK, kChannel> x;
  x.convert(raw);
  const bool fine = !__syncthreads_or(!x.fine(raw) || !(b * 0.0f == 0.0f));
  {  // B's diagonal
    float d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      d[i] = x.q[i][0] * x.k[i][0];
      if constexpr (N == 2) d[i] = fmaf(x.q[i][1], x.k[i][1], d[i]);
    }
    wave_sums8(d);
    const int row = lane / 16;
    if (lane % 16 < 2) diag[8 * wave + row / 2 * 4 + row % 2 * 2 + lane % 16] = lane % 16 ? d[1] : d[0];
  }
  // times 2^6 on both sides of a tile
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int c = 0; c < N; ++c) x.k[i][c] *= kScale, x.q[i][c] *= kScale;
  f32x4 acc[3];
#pragma unroll
  for (int level = 0; level < 5; ++level) {
    const int hh = 1 << level;
    if (level) __syncthreads();  // the last tile's operands are read
    auto put_left = [&](int row, int i) {
      const int at = channel_at<DK>(row, lane * N);
      put_split<N>(&lds.in.left_k[0][row][at], &lds.in.left_k[1][row][at], x.k[i], x.P[i]);
      put_split<N>(&lds.in.left_q[0][row][at], &lds.in.left_q[1][row][at], x.q[i], x.P[i]);
    };
    auto put_right = [&](int row, int i) {
      const int at = channel_at<DK>(row, lane * N);
      put_split<N>(&lds.in.right[0][row][at], &lds.in.right[1][row][at], x.k[i], x.X[i]);
    };
    if (hh < 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = (8 * wave + i) / (2 * hh) * hh + (i & (hh - 1));  // without bit h
        if (i & hh) put_left(row, i);
        else put_right(row, i);
      }
    } else {
      const int first = hh == 8 ? wave / 2 * 8 : wave % 2 * 8;
      if (wave & (hh / 8)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) put_left(first + i, i);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) put_right(first + i, i);
      }
    }
    if (hh < 8) x.grow(hh);
    if (hh == 4) put<N>(&total[wave][lane * N], x.P[7]);
    __syncthreads();
    if (wave / 2 == level % 2) {
      auto operand = [&](const f16(&p)[2][16][DK], int k0) {
        const int at = channel_at<DK>(lane % 16, k0 + lane / 16 * 8);
        return Pair{*reinterpret_cast<const f16x8 *>(&p[0][lane % 16][at]), *reinterpret_cast<const f16x8 *>(&p[1][lane % 16][at])};
      };
      Pair l[DK / 32][1], r[DK / 32];
#pragma unroll
      for (int k = 0; k < DK / 32; ++k) {
        l[k][0] = wave & 1 ? operand(lds.in.left_q, 32 * k) : operand(lds.in.left_k, 32 * k);
        r[k] = operand(lds.in.right, 32 * k);
      }
      f32x4 c[1] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
      product<DK / 32, 1>(l, r, c);
      acc[level / 2] = c[0];
    }
    if (hh == 8) {  // to blocks of 16
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const float t = total[wave ^ 1][lane * N + c];
          if (wave & 1) x.P[i][c] *= t;
          else x.X[i][c] *= t;
        }
    }
  }
  __syncthreads();
  // every element under the diagonal is in one level's tile
  {
    float(*to)[kC + kPad] = wave & 1 ? lds.out.B : lds.out.A;
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int hh = 1 << (2 * k + wave / 2), ic = lane / 16 * 4 + r, jc = lane % 16;
        const int i = ic / hh * 2 * hh + hh + ic % hh, j = jc / hh * 2 * hh + jc % hh;
        if (hh <= 16 && ic / hh == jc / hh) to[i][j] = acc[k][r] * (1.0f / (kScale * kScale));
      }
  }
  __syncthreads();
  auto put_out = [&](int which, int i, int j, float v) {
    f16x2 hi, lo;
    split2(v, kScale, 0.0f, 0.0f, hi, lo);
    lds.out.mat[which][i][in_order(j)] = hi[0];
    lds.out.mat[which + 1][i][in_order(j)] = lo[0];
  };
  if (wave == 0) {
    // (I + diag(beta) A)^-1 in blocks of 16: lanes 0 to 15 the columns of the first, 16 to 31 those
    // of the second by forward substitution, then -M11 N10 M00 as two small products
    const int col = lane % 16, g = lane / 16, block = g & 1;
    float t[16], most = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = 0.0f;
#pragma unroll
      for (int l = 0; l < i; ++l) v = fmaf(lds.out.A[16 * block + i][16 * block + l], t[l], v);
      t[i] = (i == col ? 1.0f : 0.0f) - beta[16 * block + i] * v;
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (else all rows are read at once, into registers)
    }
    if (lane < 32) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        (block ? lds.out.m11 : lds.out.m00)[col][i] = t[i];
        most = fmaxf(most, fabsf(t[i]));
        put_out(0, 16 * block + i, 16 * block + col, t[i]);
      }
    }
    __builtin_amdgcn_wave_barrier();
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f}, z = y, m;
    y = mfma4(*reinterpret_cast<const f32x4 *>(&lds.out.A[16 + col][4 * g]),
              *reinterpret_cast<const f32x4 *>(&lds.out.m00[col][4 * g]), y);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      y[r] *= -beta[16 + 4 * g + r];
      m[r] = lds.out.m11[4 * g + r][col];
    }
    z = mfma4(m, y, z);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      most = fmaxf(most, fabsf(z[r]));
      put_out(0, 16 + 4 * g + r, col, z[r]);
    }
    const bool large = __any(!(most < kLimit));
    if (lane == 0) lds.out.fine[0] = fine && !large;
  } else if (wave == 1) {
    float most = 0.0f;
    for (int i = lane; i < kC * kC; i += 64) {
      const int row = i / kC, c = i % kC;
      const float v = c > row ? 0.0f : c == row ? diag[row] : lds.out.B[row][c];
      most = fmaxf(most, fabsf(v));
      put_out(2, row, c, v);
    }
    const bool large = __any(!(most < kLimit));
    if (lane == 0) lds.out.fine[1] = !large;
  } else if (wave == 2) {
    // T over its diagonal blocks
#pragma unroll
    for (int k = 0; k < 4; ++k) put_out(0, 4 * k + lane / 16, 16 + lane % 16, 0.0f);
  }
  __syncthreads();
  ChunkMats &out = a.chunks[(size_t)id * a.heads_v + h];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    reinterpret_cast<u32x4 *>(out.mat)[tid + 256 * k] = reinterpret_cast<const u32x4 *>(lds.out.mat)[tid + 256 * k];
  if (tid < 2) out.fine[tid] = lds.out.fine[tid];
  if (tid < kC) out.beta[tid] = beta[tid];
}

// A sequence's chunks in turn. The first kWaves waves hold kCols columns of the state each, as the
// accumulators of DK / 16 tiles: lane l column l % 16, rows 16 kt + 4 (l / 16) + r. As the rows
// of a result are taken for the k indices of the next product (`in_order`), the state,
// beta (V - (P K) S0) and U go from result to right operand within the lane; only the left operands,
// which all waves share, pass through LDS. The four waves behind them prepare the next chunk's
// there (and its values), in the other of two buffers, and load the one after it: the
// multiplying waves wait for no load, and their stores are never waited for.
// A sequence's chunks depend on each other, so this is bound by the time of one: about 4000
// cycles of a multiplying wave, of which 84 matrix instructions are 1350 and the splitting of the
// state, V and U beside them most of the rest, and about as long in the preparing waves. 2048 tokens of 64 heads: 64 chunks, 138-143 us from run to run.
// (With f32 matrix instructions and no preparing waves 749 us; with f16 pairs 371; with loads
// ahead and barriers that wait for LDS alone 193; with the preparing waves on SIMDs of their own
// 154; with LDS pieces turned, not rows padded, and buffer loads 143; with the values and matrices
// carried by two more waves 138, the whole call 201 -> 186.) The outputs stored 4 bytes at once, by
// an exchange between neighbours, gained nothing.
template <typename E, int DK, bool kChannel, int kWaves>
__global__ __launch_bounds__(512) void k_delta_scan(DeltaArgs a, int parts) {
  constexpr int N = DK / 64, KT = DK / 16;
  using St = Stage<E, DK, kWaves>;
  __shared__ St stage[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // Workgroups go to the 8 XCDs in turn: the `parts` column blocks of one head and sequence
  // to one XCD, whose L2 then reads the rows they share once.
  const int turn = blockIdx.x / 8, part_of = turn % parts, pair = turn / parts * 8 + blockIdx.x % 8;
  if (pair >= a.heads_v * a.scanned) return;
  const int h = pair % a.heads_v;
  int seq = pair / a.heads_v;
  if (a.scanned < a.n_seq) {
    seq = uniform(nth_chunked(a, seq));
    if (seq < 0) return;
  }
  const int hk = h / (a.heads_v / a.heads_qk), g = lane / 16, m = lane % 16;
  Seq s = seq_of(a, seq);
  s = Seq{uniform(s.first), uniform(s.last)};
  if (s.last - s.first < a.chunked) return;
  const int64_t from = slot_of(a.src, seq, a.n_slots), to = slot_of(a.dst, seq, a.n_slots);
  const bool write = sole_writer(a, seq, to);
  const int chunks = chunks_of(s);
  const ChunkMats *mats = a.chunks + (size_t)first_chunk(s, seq) * a.heads_v + h;

  if (wave >= kWaves) {
    // With two multiplying waves (on the first two SIMDs) the preparing ones share the other two,
    // two on each, and the two waves that share with the multiplying ones only carry the values and
    // the matrices; else the preparing waves do both.
    constexpr int kCarriers = kWaves == 2 ? 128 : 256, kMats = 512 / kCarriers;
    const int helper = kWaves == 2 ? wave % 2 + wave / 4 * 2 : wave - kWaves;
    // lane: channels ch .. of tokens 8 g ..; as a carrier piece `part`
    const int part = tid - 256, ch = helper * (DK / 4) + m * N;
    RawSlice<E, DK, kChannel> raw;
    u32x4 mat[kMats];
    int fine[2];
    float beta;
    // 8 values of a row; kPieces such pieces are the workgroup's columns
    typedef E E8 __attribute__((ext_vector_type(8), aligned(2)));
    constexpr int kPieces = kWaves * kCols / 8;
    const uint32_t v_col = part_of * kWaves * kCols + part % kPieces * 8;
    const bool has_v = part < kC * kPieces && (int)v_col < a.dv;
    E8 val;
#pragma unroll
    for (int i = 0; i < 8; ++i) val[i] = from_f32<E>(0.0f);
    auto load = [&](int c) {
      const int t0 = s.first + c * kC;
      raw.load(a, t0, s.last - t0, h, hk, 8 * g, ch);
    };
    auto fetch = [&](int c) {
      const int t0 = s.first + c * kC;
      const ChunkMats &in = mats[(size_t)c * a.heads_v];
#pragma unroll
      for (int i = 0; i < kMats; ++i)
        mat[i] = reinterpret_cast<const u32x4 *>(in.mat)[part + kCarriers * i];
      fine[0] = in.fine[0];
      fine[1] = in.fine[1];
      beta = in.beta[part % kC];
      const uint32_t t = min(part / kPieces, s.last - t0 - 1);
      const char *vb = chunk_rows<E>(a.v, a.v_token, t0, (int64_t)h * a.dv);
      if (has_v) val = *reinterpret_cast<const E8 *>(vb + (t * (uint32_t)a.v_token + v_col) * 2);
    };
    auto carry = [&](int c) {
      St &st = stage[c & 1];
#pragma unroll
      for (int i = 0; i < kMats; ++i) {
        const int at = part + kCarriers * i;  // of 512 pieces of 8 values: 4 matrices of 32 rows of 4
        *reinterpret_cast<u32x4 *>(&st.mat[at / 128][at / 4 % 32][token_at(at / 4 % 32, at % 4 * 8)]) = mat[i];
      }
      if (part == 0) st.fine = fine[0] && fine[1];
      if (part < kC) st.beta[part] = beta;
      // infinities and NaN by their bits
      const uint16_t inf = bitcast<uint16_t>(from_f32<E>(INFINITY));
      typedef uint16_t U8 __attribute__((ext_vector_type(8)));
      const U8 bits = bitcast<U8>(val) & (uint16_t)0x7fff;
      uint16_t most = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = bits[i] > most ? bits[i] : most;
      const uint64_t bad = __ballot(most >= inf);
      uint32_t tiles = 0;
#pragma unroll
      for (int t = 0; t < kWaves; ++t) tiles |= bad & ((kPieces == 4 ? 0x3333333333333333ull : 0x0303030303030303ull) << (2 * t)) ? 1u << t : 0u;
      if (lane == 0) st.v_bad[part / 64] = tiles;
      if (part / kPieces >= s.last - (s.first + c * kC)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) val[i] = from_f32<E>(0.0f);
      }
      if (part < kC * kPieces) *reinterpret_cast<u32x4 *>(&st.v[part / kPieces][part % kPieces * 8]) = bitcast<u32x4>(val);
    };
    auto prepare = [&](int c) {
      St &st = stage[c & 1];
      const int n = s.last - (s.first + c * kC);
      if (n < kC) raw.clear(n, 8 * g);
      float d[8][N], all[N], before[N], behind[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i][j] = kChannel || j == 0 ? decay_of(raw.g[i][kChannel ? j : 0]) : d[i][0];
        float own = d[0][j];
#pragma unroll
        for (int i = 1; i < 8; ++i) own *= d[i][j];
        // products of the 8 tokens of the lane groups before and behind this one's
        const float o1 = xor_lanes<16>(own), two = own * o1, o2 = xor_lanes<32>(two);
        before[j] = kScale * ((g & 1 ? o1 : 1.0f) * (g & 2 ? o2 : 1.0f));
        behind[j] = kScale * ((g & 1 ? 1.0f : o1) * (g & 2 ? 1.0f : o2));
        all[j] = two * o2;
      }
      const int col = in_order(ch);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float k[N], q[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          before[j] *= d[i][j];
          k[j] = to_f32((E)raw.k[i][j]);
          q[j] = to_f32((E)raw.q[i][j]);
        }
        const int row = 8 * g + i, at = channel_at<DK>(row, col);
        put_split<N>(&st.pk[0][row][at], &st.pk[1][row][at], k, before);
        put_split<N>(&st.pq[0][row][at], &st.pq[1][row][at], q, before);
      }
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 4; i >= 0; i -= 4) {
          float k4[4], x4[4];
#pragma unroll
          for (int t = 3; t >= 0; --t) {
            k4[t] = to_f32((E)raw.k[i + t][j]);
            x4[t] = behind[j];
            behind[j] *= d[i + t][j];
          }
          const int at = token_at(ch + j, in_order(8 * g + i));
          put_split<4>(&st.pe[0][ch + j][at], &st.pe[1][ch + j][at], k4, x4);
        }
      if (g == 0) put<N>(&st.decay[ch], all);
    };
    // get(c): a chunk's rows on their way; set(c): into LDS
    auto run = [&](auto get, auto set) {
      if (chunks > 0) {
        get(0);
        set(0);
        if (chunks > 1) get(1);
      }
      lds_barrier();
      for (int c = 0; c < chunks; ++c) {
        if (c + 1 < chunks) {
          set(c + 1);
          if (c + 2 < chunks) get(c + 2);
        }
        lds_barrier();
      }
    };
    if constexpr (kWaves == 2) {
      if (uniform(wave) / 2 == 2) run(fetch, carry);
      else run(load, prepare);
    } else {
      run([&](int c) { load(c), fetch(c); }, [&](int c) { prepare(c), carry(c); });
    }
    return;
  }

  const int col = (part_of * kWaves + wave) * kCols + m;
  if ((part_of * kWaves + wave) * kCols >= a.dv) {  // only keeps step
    for (int c = 0; c <= chunks; ++c) lds_barrier();
    return;
  }
  const size_t head = (size_t)DK * a.dv;
  f32x4 S[KT];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      S[kt][r] = from >= 0 ? a.state[(from * a.heads_v + h) * head + (size_t)(16 * kt + 4 * g + r) * a.dv + col] : 0.0f;
  const E *v = reinterpret_cast<const E *>(a.v) + (int64_t)h * a.dv + col;
  E *out = reinterpret_cast<E *>(a.out) + (int64_t)h * a.dv + col;

  // Whether chunk c may be multiplied.
  auto fine_chunk = [&](int c) {
    const St &st = stage[c & 1];
    uint32_t bad = st.v_bad[0] | st.v_bad[1];
    if constexpr (kWaves != 2) bad |= st.v_bad[2] | st.v_bad[3];
    return uniform(st.fine && !(bad >> wave & 1)) != 0;
  };
  // Chunk c token by token in f32, where something in it is infinite, NaN or out of range, so
  // that it reaches no earlier token.
  auto by_token = [&](int c) {
    const int t0 = s.first + c * kC;
    for (int t = t0; t < min(t0 + kC, s.last); ++t) {
      const E *k = reinterpret_cast<const E *>(a.k) + (int64_t)t * a.k_token + (int64_t)hk * DK;
      const E *q = reinterpret_cast<const E *>(a.q) + (int64_t)t * a.q_token + (int64_t)hk * DK;
      const float *gp = a.g + (int64_t)t * a.g_token + (kChannel ? (int64_t)h * DK : h);
      float dot = 0.0f, o = 0.0f;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int ch = 16 * kt + 4 * g + r;
          S[kt][r] *= decay_of(gp[kChannel ? ch : 0]);
          dot = fmaf(to_f32(k[ch]), S[kt][r], dot);
        }
      dot = add_32(add_16(dot));
      const float u = a.beta[(int64_t)t * a.beta_token + h] * (to_f32(v[(int64_t)t * a.v_token]) - dot);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int ch = 16 * kt + 4 * g + r;
          S[kt][r] = fmaf(to_f32(k[ch]), u, S[kt][r]);
          o = fmaf(to_f32(q[ch]), S[kt][r], o);
        }
      o = add_32(add_16(o));
      if (g == 0) out[(int64_t)t * a.out_token] = from_f32<E>(a.scale * o);
    }
  };
  // The largest of this lane's part of its column.
  float most_state;
  auto weigh = [&] {
    most_state = 0.0f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) most_state = most_of(S[kt], most_state);
  };
  weigh();
  auto multiply = [&](int c) {
    const int t0 = s.first + c * kC, n = s.last - t0;
    const St &st = stage[c & 1];
    auto by_channel = [&](const f16(&p)[2][kC][DK], int i, int u) {
      const int at = channel_at<DK>(m, 32 * u + 8 * g);
      return Pair{*reinterpret_cast<const f16x8 *>(&p[0][16 * i + m][at]), *reinterpret_cast<const f16x8 *>(&p[1][16 * i + m][at])};
    };
    auto by_tokens = [&](const f16 *hi, const f16 *lo) {
      const int at = token_at(m, 8 * g);
      return Pair{*reinterpret_cast<const f16x8 *>(hi + at), *reinterpret_cast<const f16x8 *>(lo + at)};
    };
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int UT = KT / 2;
    // left operands are read well before their products, among the state's splitting
    Pair pk[UT][2], pq[UT][2], right[UT];
    const ColumnScale ss(most_state);
#pragma unroll
    for (int u = 0; u < UT; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) pk[u][i] = by_channel(st.pk, i, u);
#pragma unroll
    for (int u = 0; u < UT; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) pq[u][i] = by_channel(st.pq, i, u);
#pragma unroll
    for (int u = 0; u < UT; ++u) right[u] = split(S[2 * u], S[2 * u + 1], ss.to);
#pragma unroll
    for (int i = 0; i < 8 * UT; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // an LDS read,
      __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);  // four vector instructions
    }
    __builtin_amdgcn_sched_barrier(0);
    f32x4 V[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) V[i][r] = to_f32(st.v[16 * i + 4 * g + r][wave * kCols + m]);
    f32x4 X[2] = {zero, zero}, O[2] = {zero, zero}, W[2] = {zero, zero}, BU[2] = {zero, zero};
    product<UT, 2>(pk, right, X);
    product<UT, 2>(pq, right, O);
    Pair mt[1][2], mb[1][2];
    const f32x4 beta[2] = {*reinterpret_cast<const f32x4 *>(&st.beta[4 * g]), *reinterpret_cast<const f32x4 *>(&st.beta[16 + 4 * g])};
#pragma unroll
    for (int i = 0; i < 2; ++i) mt[0][i] = by_tokens(st.mat[0][16 * i + m], st.mat[1][16 * i + m]);
#pragma unroll
    for (int i = 0; i < 2; ++i) mb[0][i] = by_tokens(st.mat[2][16 * i + m], st.mat[3][16 * i + m]);
    const float cs = ss.back / kScale;
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) X[i][r] = beta[i][r] * fmaf(-cs, X[i][r], V[i][r]);
      most = most_of(X[i], most);
    }
    const ColumnScale sx(most);
    const Pair x[1] = {split(X[0], X[1], sx.to)};
    product<1, 2>(mt, x, W);
    Pair pe[1][KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) pe[0][kt] = by_tokens(st.pe[0][16 * kt + m], st.pe[1][16 * kt + m]);
    most = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) W[i][r] *= sx.back / kScale;
      most = most_of(W[i], most);
    }
    const ColumnScale su(most);
    const Pair u[1] = {split(W[0], W[1], su.to)};
    const float cu = su.back / kScale;
    product<1, 2>(mb, u, BU);
    f32x4 add[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) add[kt] = zero;
    product<1, KT>(pe, u, add);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const f32x4 d = *reinterpret_cast<const f32x4 *>(&st.decay[16 * kt + 4 * g]);
#pragma unroll
      for (int r = 0; r < 4; ++r) S[kt][r] = fmaf(cu, add[kt][r], d[r] * S[kt][r]);
    }
    weigh();
    char *ob = const_cast<char *>(chunk_rows<E>(a.out, a.out_token, t0, (int64_t)h * a.dv));
    const uint32_t os = (uint32_t)a.out_token * 2, oo = 4 * g * os + col * 2;
    E o[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[i][r] = from_f32<E>(a.scale * fmaf(cs, O[i][r], cu * BU[i][r]));
    if (n >= kC) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) *reinterpret_cast<E *>(ob + (oo + (16 * i + r) * os)) = o[i][r];
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * i + 4 * g + r < n) *reinterpret_cast<E *>(ob + (oo + (16 * i + r) * os)) = o[i][r];
    }
  };
  lds_barrier();
  // the rare chunks outside the loop over the others, whose registers and waits they would shape
  for (int c = 0; c < chunks; ++c, lds_barrier()) {
    for (; c < chunks && fine_chunk(c); ++c, lds_barrier()) multiply(c);
    if (c == chunks) break;
    by_token(c);
    weigh();
  }
  if (write)
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        a.state[(to * a.heads_v + h) * head + (size_t)(16 * kt + 4 * g + r) * a.dv + col] = S[kt][r];
}

// f(DK, channel) as compile-time values.
template <typename F>
void with_form(int dk, bool channel, F &&f) {
  if (dk == 64) {
    if (channel) f(std::integral_constant<int, 64>{}, std::true_type{});
    else f(std::integral_constant<int, 64>{}, std::false_type{});
  } else {
    if (channel) f(std::integral_constant<int, 128>{}, std::true_type{});
    else f(std::integral_constant<int, 128>{}, std::false_type{});
  }
}

exl3_status check_config(const exl3_delta_config *c) {
  using exl3h::fail;
  if (!c) return fail(EXL3_ERR_INVALID, "exl3_delta_rule: null config");
  if (c->dtype != EXL3_ST_F16 && c->dtype != EXL3_ST_BF16)
    return fail(EXL3_ERR_UNSUPPORTED, "exl3_delta_rule: dtype must be f16 or bf16");
  if (c->heads_qk < 1 || c->heads_v < 1 || c->heads_v > 4096 || c->heads_v % c->heads_qk)
    return fail(EXL3_ERR_INVALID, "exl3_delta_rule: heads_v (at most 4096) must be a multiple of heads_qk");
  if (c->dk != 64 && c->dk != 128) return fail(EXL3_ERR_UNSUPPORTED, "exl3_delta_rule: dk must be 64 or 128");
  if (c->dv < 16 || c->dv > 256 || c->dv % 16)
    return fail(EXL3_ERR_UNSUPPORTED, "exl3_delta_rule: dv must be a multiple of 16 up to 256");
  return EXL3_OK;
}

// Which sequences go in chunks. A sequence does from 16 tokens on: chunks against steps at 8, 16 and 24 tokens each, in us: one sequence of 64 heads 17.7
// against 11.0, 17.6 / 18.0, 17.8 / 25.0; 16 of them 82 / 53, 83 / 88, 85 / 122; 64 sequences of 8
// heads 48 / 30, 48 / 49, 51 / 68. With `starts` the host does not know the lengths, only
// how many tokens there are: under 64 past one a sequence and under 16 a sequence all go in
// steps, from 64 a sequence on all in chunks, and between them each by its own length.
// All steps, all chunks and each by its own, in us for 64 heads: 256 sequences of one token
// beside one of 2048 3201, 1370, 690; 64 beside one of 128 259, 316, 126; 8 beside one of 512
// 439, 105, 88; 1 to 1001 tokens 830, 160, 160. The others' launches cost 64 sequences of 4
// 142 against 136, 16 of them in 16 heads 17 against 14.
constexpr int kChunked = 16, kFewTokens = 64, kManyTokens = 64;
enum Form { kSteps, kChunks, kBoth };
Form form_of(int64_t tokens, int64_t n_seq, bool starts) {
  if (!starts || n_seq == 1) return tokens >= kChunked * n_seq ? kChunks : kSteps;
  if (tokens >= kManyTokens * n_seq) return kChunks;
  return tokens >= kChunked * n_seq || tokens - n_seq >= kFewTokens ? kBoth : kSteps;
}
int64_t chunk_ids(int64_t tokens, int64_t n_seq) { return tokens / kC + n_seq; }
size_t chunk_bytes(const exl3_delta_config *c, int64_t tokens, int64_t n_seq, bool starts) {
  return n_seq && form_of(tokens, n_seq, starts) != kSteps
             ? exl3h::align_up((size_t)chunk_ids(tokens, n_seq) * c->heads_v * sizeof(ChunkMats), 256) : 0;
}

bool bad_counts(int64_t tokens, int64_t n_seq) {
  return tokens < 0 || tokens > ((int64_t)1 << 27) || n_seq < 0 || n_seq > 65535;
}
// Heads of all sequences: a launch holds 2^32 threads in a dimension, the scan four workgroups
// of 512 a head.
bool too_many(const exl3_delta_config *c, int64_t n_seq) { return c->heads_v * n_seq > (1 << 20); }

}  // namespace

using namespace exl3h;

extern "C" {

size_t exl3_delta_workspace_size(const exl3_delta_config *cfg, int64_t tokens, int64_t n_seq) {
  if (check_config(cfg) || bad_counts(tokens, n_seq) || too_many(cfg, n_seq)) return 0;
  return std::max(chunk_bytes(cfg, tokens, n_seq, true), chunk_bytes(cfg, tokens, n_seq, false));
}

exl3_status exl3_delta_rule(const exl3_delta_config *cfg, const exl3_delta_rows *x, int64_t tokens,
                            const int32_t *starts, int64_t n_seq, float *state, int64_t n_slots, const int32_t *src,
                            const int32_t *dst, void *workspace, size_t workspace_bytes, exl3_stream_t stream) {
  exl3_status rc = check_config(cfg);
  if (rc) return rc;
  if (bad_counts(tokens, n_seq))
    return fail(EXL3_ERR_INVALID, "exl3_delta_rule: at most 2^27 tokens of at most 65,535 sequences");
  if (too_many(cfg, n_seq))
    return fail(EXL3_ERR_INVALID, "exl3_delta_rule: at most 2^20 value heads over all sequences");
  if (n_seq == 0) return EXL3_OK;
  if (!starts && tokens % n_seq)
    return fail(EXL3_ERR_INVALID, "exl3_delta_rule: without starts the tokens must divide into the sequences");
  if (!x) return fail(EXL3_ERR_INVALID, "exl3_delta_rule: null rows");
  if (n_slots < 1 || n_slots > ((int64_t)1 << 31) - 1)
    return fail(EXL3_ERR_INVALID, "exl3_delta_rule: bad slot count");
  if (!state || (tokens && (!x->q || !x->k || !x->v || !x->g || !x->beta || !x->out)))
    return fail(EXL3_ERR_INVALID, "exl3_delta_rule: null argument");
  const int64_t qk = (int64_t)cfg->heads_qk * cfg->dk, vo = (int64_t)cfg->heads_v * cfg->dv;
  const int64_t gs = cfg->heads_v * (cfg->channel_decay ? (int64_t)cfg->dk : 1);
  const int64_t strides[6][2] = {{x->q_token, qk}, {x->k_token, qk}, {x->v_token, vo},
                                 {x->out_token, vo}, {x->g_token, gs}, {x->beta_token, cfg->heads_v}};
  for (const auto &s : strides)
    // (under 2^24 elements, a chunk's rows lie within 32-bit offsets)
    if (tokens > 1 && (s[0] < s[1] || s[0] >= ((int64_t)1 << 24)))
      return fail(EXL3_ERR_INVALID, "exl3_delta_rule: a token stride is smaller than a token's heads, or 2^24 or more");
  if ((reinterpret_cast<uintptr_t>(x->q) | reinterpret_cast<uintptr_t>(x->k) | reinterpret_cast<uintptr_t>(x->v) |
       reinterpret_cast<uintptr_t>(x->out)) % 2 ||
      (reinterpret_cast<uintptr_t>(x->g) | reinterpret_cast<uintptr_t>(x->beta) | reinterpret_cast<uintptr_t>(starts) |
       reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) % 4 ||
      reinterpret_cast<uintptr_t>(state) % 16)
    return fail(EXL3_ERR_INVALID, "exl3_delta_rule: rows must be 2-byte, f32 and i32 arguments 4-byte, the state 16-byte aligned");
  // bytes from a first row's start to past a last row's end
  auto span = [&](int i, size_t size) { return tokens ? ((tokens - 1) * strides[i][0] + strides[i][1]) * size : 0; };
  const size_t state_bytes = (size_t)n_slots * cfg->heads_v * cfg->dk * cfg->dv * 4;
  const void *const rows[6] = {x->q, x->k, x->v, x->out, x->g, x->beta};
  for (int i = 0; i < 6; ++i)
    if ((i != 3 && spans_meet(x->out, span(3, 2), rows[i], span(i, i < 4 ? 2 : 4))) ||
        spans_meet(state, state_bytes, rows[i], span(i, i < 4 ? 2 : 4)))
      return fail(EXL3_ERR_INVALID, "exl3_delta_rule: out and state must not overlap the call's other rows");
  const Form form = form_of(tokens, n_seq, starts != nullptr);
  const size_t need = chunk_bytes(cfg, tokens, n_seq, starts != nullptr);
  if (need && (!workspace || workspace_bytes < need))
    return fail(EXL3_ERR_WORKSPACE, "exl3_delta_rule: workspace too small: need " + std::to_string(need) + " bytes");
  if (need && reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(EXL3_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  for (int i = 0; i < 7; ++i)
    if (need && (i < 6 ? spans_meet(workspace, need, rows[i], span(i, i < 4 ? 2 : 4)) : spans_meet(workspace, need, state, state_bytes)))
      return fail(EXL3_ERR_INVALID, "exl3_delta_rule: the workspace must not overlap rows or state");
  DeltaArgs a = {};
  a.q = x->q;
  a.k = x->k;
  a.v = x->v;
  a.g = x->g;
  a.beta = x->beta;
  a.out = x->out;
  a.q_token = x->q_token;
  a.k_token = x->k_token;
  a.v_token = x->v_token;
  a.g_token = x->g_token;
  a.beta_token = x->beta_token;
  a.out_token = x->out_token;
  a.tokens = (int32_t)tokens;
  a.n_seq = (int32_t)n_seq;
  a.heads_qk = cfg->heads_qk;
  a.heads_v = cfg->heads_v;
  a.dv = cfg->dv;
  a.scale = cfg->scale;
  a.starts = starts;
  a.state = state;
  a.n_slots = n_slots;
  a.src = src;
  a.dst = dst ? dst : src;
  a.chunks = reinterpret_cast<ChunkMats *>(workspace);
  a.chunked = form == kSteps ? INT32_MAX : form == kChunks ? 0 : kChunked;
  a.scanned = (int32_t)(form == kBoth ? std::min(n_seq, tokens / kChunked) : n_seq);
  a.words = (reinterpret_cast<uintptr_t>(x->q) | reinterpret_cast<uintptr_t>(x->k)) % 4 == 0 && (x->q_token | x->k_token) % 2 == 0;
  with_elem16(cfg->dtype, [&](auto e) {
    using E = decltype(e);
    with_form(cfg->dk, cfg->channel_decay != 0, [&](auto dk, auto channel) {
      constexpr int DK = decltype(dk)::value;
      constexpr bool kChannel = decltype(channel)::value;
      const hipStream_t st = stream_of(stream);
      if (form != kSteps) {
        k_delta_chunk<E, DK, kChannel><<<dim3((unsigned)chunk_ids(tokens, n_seq), (unsigned)cfg->heads_v), 256, 0, st>>>(a);
        // Two column blocks a workgroup where all workgroups then have a CU of their own, else four,
        // which share the preparation: a 2048-token sequence of 64 heads 169 against 190 us, 7
        // sequences of up to 1001 tokens of 32 heads 119 against 94 us (both before the
        // preparing waves moved to SIMDs of their own, which took 16 us off the first).
        auto scan = [&](auto waves) {
          constexpr int kWaves = decltype(waves)::value;
          const int parts = (cfg->dv / kCols + kWaves - 1) / kWaves;
          const unsigned blocks = (unsigned)(((int64_t)cfg->heads_v * a.scanned + 7) / 8 * 8 * parts);
          k_delta_scan<E, DK, kChannel, kWaves><<<blocks, 512, 0, st>>>(a, parts);
        };
        if ((cfg->dv / kCols + 1) / 2 * (int64_t)cfg->heads_v * a.scanned <= 256) scan(std::integral_constant<int, 2>{});
        else scan(std::integral_constant<int, 4>{});
      }
      if (form != kChunks) {
        const dim3 grid((unsigned)((cfg->dv / kCols + 3) / 4), (unsigned)cfg->heads_v, (unsigned)n_seq);
        k_delta_step<E, DK, kChannel><<<grid, 256, 0, st>>>(a);
      }
    });
  });
  EXL3_LAUNCHED("k_delta");
  return EXL3_OK;
}

}  // extern "C"
