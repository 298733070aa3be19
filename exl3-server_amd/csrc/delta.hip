// The gated delta rule over a batch of sequences of any lengths (gfx950).
//
// A head's state S (dk, dv) is f32. For each token, with a = exp(g) (one decay for the head,
// or one per key channel):
//   S <- diag(a) S;  u = beta (v - S^T k);  S <- S + k u^T;  out = scale S^T q
//
//  k_delta_step   token by token: the state in registers from its slot to its slot.
#include <hip/hip_runtime.h>

#include <string>

#include "elem.hpp"
#include "exl3_device.hpp"
#include "exl3_internal.hpp"
#include "exl3_moe.h"

using namespace exl3d;
using namespace exl3e;

namespace {

constexpr int kCols = 16;  // state columns of a wave

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
  bool met = false;
  for (int j = threadIdx.x; j < a.n_seq; j += blockDim.x)
    if (j != i) met |= slot_of(a.src, j, a.n_slots) == slot || slot_of(a.dst, j, a.n_slots) == slot;
  return !__syncthreads_or(met) && slot >= 0;
}

// Sum over the 16 lanes of a wave that hold the same columns (lane / 4).
__device__ __forceinline__ f32x4 sum_rows(f32x4 v) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float x = v[c];
    x += xor_lanes<4>(x);
    x += xor_lanes<8>(x);
    x += xor_lanes<16>(x);
    x += xor_lanes<32>(x);
    v[c] = x;
  }
  return v;
}

// A wave holds kCols columns of the state: lane l the columns 4 (l % 4).. and the DK / 16
// rows from (l / 4) DK / 16.
template <typename E, int DK, bool kChannel>
__global__ __launch_bounds__(256) void k_delta_step(DeltaArgs a) {
  constexpr int R = DK / 16;
  const int lane = threadIdx.x & 63, seq = blockIdx.z, h = blockIdx.y, hk = h / (a.heads_v / a.heads_qk);
  const int64_t from = slot_of(a.src, seq, a.n_slots), to = slot_of(a.dst, seq, a.n_slots);
  const bool write = sole_writer(a, seq, to);
  const int block = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (block * kCols >= a.dv) return;
  const Seq s = seq_of(a, seq);
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
  for (int64_t t = s.first; t < s.last; ++t) {
    float kk[R], qq[R], decay[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      kk[r] = to_f32(k[t * a.k_token + r]);
      qq[r] = to_f32(q[t * a.q_token + r]);
      decay[r] = g[t * a.g_token + (kChannel ? r : 0)];
    }
    const float beta = a.beta[t * a.beta_token + h];
    f32x4 vv;
#pragma unroll
    for (int c = 0; c < 4; ++c) vv[c] = to_f32(v[t * a.v_token + c]);
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

bool bad_counts(int64_t tokens, int64_t n_seq) {
  return tokens < 0 || tokens > ((int64_t)1 << 30) || n_seq < 0 || n_seq > 65535;
}

}  // namespace

using namespace exl3h;

extern "C" {

size_t exl3_delta_workspace_size(const exl3_delta_config *cfg, int64_t tokens, int64_t n_seq) {
  if (check_config(cfg) || bad_counts(tokens, n_seq)) return 0;
  return 0;
}

exl3_status exl3_delta_rule(const exl3_delta_config *cfg, const exl3_delta_rows *x, int64_t tokens,
                            const int32_t *starts, int64_t n_seq, float *state, int64_t n_slots, const int32_t *src,
                            const int32_t *dst, void *workspace, size_t workspace_bytes, exl3_stream_t stream) {
  exl3_status rc = check_config(cfg);
  if (rc) return rc;
  if (bad_counts(tokens, n_seq))
    return fail(EXL3_ERR_INVALID, "exl3_delta_rule: at most 2^30 tokens of at most 65,535 sequences");
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
    if (tokens > 1 && (s[0] < s[1] || s[0] > ((int64_t)1 << 31)))
      return fail(EXL3_ERR_INVALID, "exl3_delta_rule: a token stride is smaller than a token's heads");
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
  with_elem16(cfg->dtype, [&](auto e) {
    using E = decltype(e);
    with_form(cfg->dk, cfg->channel_decay != 0, [&](auto dk, auto channel) {
      const dim3 grid((unsigned)((cfg->dv / kCols + 3) / 4), (unsigned)cfg->heads_v, (unsigned)n_seq);
      k_delta_step<E, decltype(dk)::value, decltype(channel)::value><<<grid, 256, 0, stream_of(stream)>>>(a);
    });
  });
  EXL3_LAUNCHED("k_delta_step");
  return EXL3_OK;
}

}  // extern "C"
