// linear.hip -- linear attention with a decay for each head, on gfx950.  The
// reference has no counterpart; its closest relative here is the Mamba-2 SSD
// (ssd.hip, mamba.hip), whose decays depend on the token and which has no form for
// single tokens.
//
//   q [B, T, G, H, D], k [B, T, G, D], v [B, T, G, E], log_decay [G, H] fp32,
//   state [B, G, H, D, E] fp32.  For every (b, g, h), with a = exp(log_decay[g, h]):
//     S_t = a S_(t-1) + k_t v_t^T,   out_t = scale S_t^T q_t,   S_(-1) = state or 0;
//   sequence b has c = clamp(counts[b], 0, T) tokens (all T without counts), state_out
//   is S_(c-1), and out's rows t >= c are left as they are.
#include "common.h"

#include <cmath>

namespace {

struct LinearParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const float* g;        // log decays
  const float* state;
  const int* counts;
  uint16_t* out;
  float* state_out;
  int B, G, H, D, E, T;
  float scale;
};

// exp(n g) in 64 bits; a head without memory (g = -inf) keeps its own token, n = 0
LOOM_DEV double decay_pow(float g, int n) {
  return exp((double)n * (double)(g < -1e30f ? -1e30f : g));
}

// One factor as a sum of two floats: a rounded decay near 1, applied over and
// over, would be off by its rounding times the tokens that a head remembers.
struct Decay {
  float hi, lo;
};
LOOM_DEV Decay split_decay(double x) {
  const float hi = (float)x;
  return Decay{hi, (float)(x - (double)hi)};
}
LOOM_DEV float decayed(float s, const Decay& a) { return __builtin_fmaf(s, a.hi, s * a.lo); }

// Token by token: 16 columns of one state to a workgroup, 16 threads to a column.
template <bool F16>
__global__ void __launch_bounds__(256) linear_token_kernel(LinearParams p) {
  const int sub = threadIdx.x & 15, e = blockIdx.y * 16 + (threadIdx.x >> 4);
  const int GH = p.G * p.H;
  const int b = blockIdx.x / GH, gh = blockIdx.x % GH, g = gh / p.H;
  const int c = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  const Decay a = split_decay(decay_pow(p.g[gh], 1));
  const int64_t s0 = (int64_t)blockIdx.x * p.D * p.E + e;
  const bool in = e < p.E;
  float s[16];
  for (int i = 0; i < 16; ++i) {
    const int d = sub + 16 * i;
    s[i] = in && d < p.D && p.state ? p.state[s0 + (int64_t)d * p.E] : 0.f;
  }
  for (int t = 0; t < c; ++t) {
    const int64_t tok = (int64_t)b * p.T + t;
    const uint16_t* q = p.q + (tok * GH + gh) * p.D;
    const uint16_t* k = p.k + (tok * p.G + g) * p.D;
    const float v = in ? lo16<F16>(p.v[(tok * p.G + g) * p.E + e]) : 0.f;
    float o = 0.f;
    for (int i = 0; i < 16; ++i) {
      const int d = sub + 16 * i;
      if (d < p.D) {
        s[i] = __builtin_fmaf(lo16<F16>(k[d]), v, decayed(s[i], a));
        o += lo16<F16>(q[d]) * s[i];
      }
    }
    for (int m = 8; m >= 1; m >>= 1) o += __shfl_xor(o, m);
    if (in && sub == 0) p.out[(tok * GH + gh) * p.E + e] = (uint16_t)cvt16<F16>(o * p.scale);
  }
  for (int i = 0; i < 16; ++i) {
    const int d = sub + 16 * i;
    if (in && d < p.D) p.state_out[s0 + (int64_t)d * p.E] = s[i];
  }
}

template <bool F16>
int linear_impl(const char* what, const void* q, const void* k, const void* v,
                const void* log_decay, const void* state, const void* counts, void* out,
                void* state_out, void* workspace, size_t workspace_bytes, int64_t B, int64_t G,
                int64_t H, int64_t D, int64_t E, int64_t T, float scale, void* stream, char* err,
                size_t errlen) {
  if (!q || !k || !v || !log_decay || !out || !state_out)
    return loom_fail(err, errlen, LOOM_EINVAL, "%s: null tensor pointer", what);
  if (B <= 0 || G <= 0 || H <= 0 || D <= 0 || E <= 0 || T <= 0)
    return loom_fail(err, errlen, LOOM_EINVAL, "%s: extents must be positive", what);
  if (!(scale > 0.f) || !std::isfinite(scale))
    return loom_fail(err, errlen, LOOM_EINVAL, "%s: scale must be finite and positive (got %g)",
                     what, (double)scale);
  if (D % 8 != 0 || D > 256 || E % 8 != 0 || E > 256)
    return loom_fail(err, errlen, LOOM_EUNSUP,
                     "%s: key dim %lld, value dim %lld not built (multiples of 8 up to 256)", what,
                     (long long)D, (long long)E);
  if (T > (1 << 29) || !loom_prod_le({B, G, H}, 1 << 20))
    return loom_fail(err, errlen, LOOM_EINVAL, "%s: problem too large", what);
  auto aligned4 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(state) ||
      !aligned16(state_out) || !aligned4(log_decay) || !aligned4(counts))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "%s: tensors must be 16-byte aligned (log_decay and counts 4-byte)", what);
  const size_t need = loom_hip_linear_attention_workspace_bytes(B, G, H, D, E, T);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "%s: workspace needs %zu bytes (16-byte aligned), got %zu", what, need,
                     workspace_bytes);
  // state_out on state is safe: a state is read before, and by the threads that write it
  const int64_t tokens = B * T * G * 2, states = B * G * H * D * E * 4;
  const LoomSpan in[] = {{q, tokens * H * D}, {k, tokens * D}, {v, tokens * E},
                         {log_decay, G * H * 4}, {counts, B * 4},
                         {state == state_out ? nullptr : state, states}},
                 outs[] = {{out, tokens * H * E}, {state_out, states},
                           {need ? workspace : nullptr, (int64_t)need}};
  if (loom_outputs_overlap(in, outs))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "%s: outputs and the workspace must not overlap the other tensors or each "
                     "other (but state_out may be state)",
                     what);
  LinearParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.g = static_cast<const float*>(log_decay);
  p.state = static_cast<const float*>(state);
  p.counts = static_cast<const int*>(counts);
  p.out = static_cast<uint16_t*>(out);
  p.state_out = static_cast<float*>(state_out);
  p.B = (int)B;
  p.G = (int)G;
  p.H = (int)H;
  p.D = (int)D;
  p.E = (int)E;
  p.T = (int)T;
  p.scale = scale;
  if (loom_validate_only()) return loom_ok(err, errlen);
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL((linear_token_kernel<F16>),
                     dim3((unsigned)(B * G * H), (unsigned)cdiv64(E, 16)), dim3(256), 0, st, p);
  return loom_check_launch(err, errlen, what);
}

}  // namespace

extern "C" {

size_t loom_hip_linear_attention_workspace_bytes(int64_t B, int64_t G, int64_t H, int64_t D,
                                                 int64_t E, int64_t T) {
  return 0;
}

int loom_hip_linear_attention(const void* q, const void* k, const void* v, const void* log_decay,
                              const void* state, const void* counts, void* out, void* state_out,
                              void* workspace, size_t workspace_bytes, int64_t B, int64_t G,
                              int64_t H, int64_t D, int64_t E, int64_t T, float scale,
                              void* stream, char* err, size_t errlen) {
  return linear_impl<false>("linear_attention", q, k, v, log_decay, state, counts, out, state_out,
                            workspace, workspace_bytes, B, G, H, D, E, T, scale, stream, err,
                            errlen);
}
int loom_hip_linear_attention_f16(const void* q, const void* k, const void* v,
                                  const void* log_decay, const void* state, const void* counts,
                                  void* out, void* state_out, void* workspace,
                                  size_t workspace_bytes, int64_t B, int64_t G, int64_t H,
                                  int64_t D, int64_t E, int64_t T, float scale, void* stream,
                                  char* err, size_t errlen) {
  return linear_impl<true>("linear_attention", q, k, v, log_decay, state, counts, out, state_out,
                           workspace, workspace_bytes, B, G, H, D, E, T, scale, stream, err,
                           errlen);
}

int loom_hip_linear_attention_step(const void* q, const void* k, const void* v,
                                   const void* log_decay, void* state, const void* counts,
                                   void* out, int64_t B, int64_t G, int64_t H, int64_t D,
                                   int64_t E, float scale, void* stream, char* err,
                                   size_t errlen) {
  return linear_impl<false>("linear_attention_step", q, k, v, log_decay, state, counts, out, state,
                            nullptr, 0, B, G, H, D, E, 1, scale, stream, err, errlen);
}
int loom_hip_linear_attention_step_f16(const void* q, const void* k, const void* v,
                                       const void* log_decay, void* state, const void* counts,
                                       void* out, int64_t B, int64_t G, int64_t H, int64_t D,
                                       int64_t E, float scale, void* stream, char* err,
                                       size_t errlen) {
  return linear_impl<true>("linear_attention_step", q, k, v, log_decay, state, counts, out, state,
                           nullptr, 0, B, G, H, D, E, 1, scale, stream, err, errlen);
}

}  // extern "C"
