// cache_decode.hip -- one decoding step over caches of different lengths, with
// an optional prefix that all sequences share and the keys' attention weights
// gathered, on gfx950.  The reference has no counterpart; its @flash_decode
// (decode.hip) is the step of one KV head over caches of one length.
//
//   q, out [B, G, H, D]; prefix_k [G, D, P], prefix_v [G, P, D]; k [B, G, D, S]
//   (keys transposed), v [B, G, S, D]; lens [B]: sequence b holds
//   n = clamp(lens[b], 0, S) keys.  For every row (b, g, h), over the P prefix
//   keys of head g and the n keys of (b, g) together:
//     s_j = scale q . key_j, p_j = exp(s_j - max s) / sum exp(s - max s),
//     out = sum_j p_j v_j;
//     weights_out[b, g, j] = weights[b, g, j] + sum_h p_j for the own keys.
//   A row without keys is zero.
#include "common.h"

#include <cmath>

namespace {

struct StepParams {
  const uint16_t* pk;
  const uint16_t* pv;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  const int* lens;
  const float* w;
  float* w_out;
  uint16_t* out;
  float* score;   // [B G H, P + S], log2 domain
  float* ml;      // [B G H, 2]: maximum and sum of a row
  int B, G, H, D, P, S;
  float c2;       // scale * log2(e)
};

constexpr int kThreads = 256;

// One workgroup per row (b, g, h): the scores (a thread per key), their
// maximum and sum, then the values' weighted sum (a thread per d).
template <bool F16>
__global__ void __launch_bounds__(kThreads) cache_row_kernel(StepParams p) {
  __shared__ float s_q[256], s_red[kThreads / 64], s_o[kThreads];
  const int64_t row = blockIdx.x;
  const int64_t bg = row / p.H;
  const int b = (int)(bg / p.G), g = (int)(bg % p.G);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int D = p.D, P = p.P, n = min(max(p.lens[b], 0), p.S), N = P + n;
  const uint16_t* const pk = p.pk + (int64_t)g * D * P;
  const uint16_t* const pv = p.pv + (int64_t)g * P * D;
  const uint16_t* const k = p.k + bg * D * p.S;
  const uint16_t* const v = p.v + bg * p.S * D;
  float* const sc = p.score + row * (P + p.S);
  if (tid < D) s_q[tid] = lo16<F16>(p.q[row * D + tid]);
  __syncthreads();
  float m = -INFINITY;
  for (int j = tid; j < N; j += kThreads) {
    float s = 0.f;
    if (j < P)
      for (int d = 0; d < D; ++d) s += s_q[d] * lo16<F16>(pk[(int64_t)d * P + j]);
    else
      for (int d = 0; d < D; ++d) s += s_q[d] * lo16<F16>(k[(int64_t)d * p.S + j - P]);
    s *= p.c2;
    sc[j] = s;
    m = fmaxf(m, s);
  }
  m = wave_max(m);
  if (lane == 0) s_red[wave] = m;
  __syncthreads();
  for (int x = 0; x < kThreads / 64; ++x) m = fmaxf(m, s_red[x]);
  const float base = m == -INFINITY ? 0.f : m;
  __syncthreads();
  float l = 0.f;
  for (int j = tid; j < N; j += kThreads) l += exp2f(sc[j] - base);
  l = wave_sum(l);
  if (lane == 0) s_red[wave] = l;
  __syncthreads();
  l = 0.f;
  for (int x = 0; x < kThreads / 64; ++x) l += s_red[x];
  const float inv = l != 0.f ? 1.f / l : 0.f;
  if (tid == 0) {
    p.ml[2 * row] = base;
    p.ml[2 * row + 1] = inv;
  }
  for (int d0 = 0; d0 < D; d0 += 64) {
    const int d = d0 + lane;
    float o = 0.f;
    if (d < D)
      for (int j = wave; j < N; j += kThreads / 64) {
        const float e = exp2f(sc[j] - base);
        const uint32_t x = j < P ? pv[(int64_t)j * D + d] : v[(int64_t)(j - P) * D + d];
        o += e * lo16<F16>(x);
      }
    s_o[tid] = o;
    __syncthreads();
    if (wave == 0 && d < D) {
      for (int x = 1; x < kThreads / 64; ++x) o += s_o[x * 64 + lane];
      p.out[row * D + d] = (uint16_t)cvt16<F16>(o * inv);
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(256) cache_weight_kernel(StepParams p) {
  const int64_t bg = blockIdx.y;
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= min(max(p.lens[bg / p.G], 0), p.S)) return;
  float a = 0.f;
  for (int h = 0; h < p.H; ++h) {
    const int64_t row = bg * p.H + h;
    a += exp2f(p.score[row * (p.P + p.S) + p.P + j] - p.ml[2 * row]) * p.ml[2 * row + 1];
  }
  p.w_out[bg * p.S + j] = p.w[bg * p.S + j] + a;
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <bool F16>
int cache_decode_impl(const void* prefix_k, const void* prefix_v, const void* k, const void* v,
                      const void* q, const void* lens, const void* weights, void* weights_out,
                      void* out, void* workspace, size_t workspace_bytes, int64_t B, int64_t G,
                      int64_t H, int64_t D, int64_t P, int64_t S, float scale, void* stream,
                      char* err, size_t errlen) {
  if (!k || !v || !q || !lens || !out)
    return loom_fail(err, errlen, LOOM_EINVAL, "cache_decode: null tensor pointer");
  if (B <= 0 || G <= 0 || H <= 0 || D <= 0 || S <= 0 || P < 0)
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_decode: extents must be positive (P may be 0)");
  if ((P > 0) != (prefix_k != nullptr) || (P > 0) != (prefix_v != nullptr))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_decode: prefix_k and prefix_v go with P > 0, null with P == 0");
  if ((weights != nullptr) != (weights_out != nullptr))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_decode: weights and weights_out are given together or not at all");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_decode: scale must be finite and positive (got %g)", (double)scale);
  if (D % 8 != 0 || D > 256)
    return loom_fail(err, errlen, LOOM_EUNSUP,
                     "cache_decode: head_dim %lld not built (a multiple of 8 up to 256)",
                     (long long)D);
  if (S > (1 << 30) || P > (1 << 30) || !loom_prod_le({B, G}, 65535) ||
      !loom_prod_le({B, G, H}, 1 << 24) || !loom_prod_le({B, G, S, D}, (int64_t)1 << 50) ||
      !loom_prod_le({G, P, D}, (int64_t)1 << 50))
    return loom_fail(err, errlen, LOOM_EINVAL, "cache_decode: problem too large");
  // a capacity or prefix that is not a multiple of 8 takes buffer descriptors,
  // which address one (b, g)'s keys in 32 bits
  if ((S % 8 != 0 && !loom_prod_le({D, S, 2}, 0x7fffffffll)) ||
      (P % 8 != 0 && !loom_prod_le({D, P, 2}, 0x7fffffffll)))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_decode: D*S or D*P too large for an extent that is not a multiple of 8");
  if (!aligned(k, S % 8 == 0 ? 16 : 2) || !aligned(prefix_k, P % 8 == 0 ? 16 : 2) ||
      !aligned16(v) || !aligned16(prefix_v) || !aligned16(q) || !aligned16(out) ||
      !aligned(lens, 4) || !aligned(weights, 4) || !aligned(weights_out, 4))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_decode: tensors must be 16-byte aligned (k and prefix_k 2-byte when "
                     "their extent is not a multiple of 8; lens and weights 4-byte)");
  const uintptr_t w0 = reinterpret_cast<uintptr_t>(weights);
  const uintptr_t w1 = reinterpret_cast<uintptr_t>(weights_out);
  if (w0 != w1 && w0 < w1 + (uint64_t)(B * G * S * 4) && w1 < w0 + (uint64_t)(B * G * S * 4))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_decode: weights_out is weights itself or does not overlap it");
  const size_t need = loom_hip_cache_decode_workspace_bytes(B, G, H, D, P, S, weights != nullptr);
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_decode: workspace needs %zu bytes (16-byte aligned), got %zu", need,
                     workspace_bytes);
  StepParams p{};
  p.pk = static_cast<const uint16_t*>(prefix_k);
  p.pv = static_cast<const uint16_t*>(prefix_v);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q = static_cast<const uint16_t*>(q);
  p.lens = static_cast<const int*>(lens);
  p.w = static_cast<const float*>(weights);
  p.w_out = static_cast<float*>(weights_out);
  p.out = static_cast<uint16_t*>(out);
  p.ml = static_cast<float*>(workspace);
  p.score = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                     align256((size_t)B * G * H * 8));
  p.B = (int)B;
  p.G = (int)G;
  p.H = (int)H;
  p.D = (int)D;
  p.P = (int)P;
  p.S = (int)S;
  p.c2 = scale * 1.4426950408889634f;
  if (loom_validate_only()) return loom_ok(err, errlen);
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(cache_row_kernel<F16>, dim3((unsigned)(B * G * H)), dim3(kThreads), 0, st, p);
  int rc = loom_check_launch(err, errlen, "cache_decode");
  if (rc || !weights) return rc;
  hipLaunchKernelGGL(cache_weight_kernel, dim3((unsigned)cdiv64(S, 256), (unsigned)(B * G)),
                     dim3(256), 0, st, p);
  return loom_check_launch(err, errlen, "cache_decode (weights)");
}

}  // namespace

extern "C" {

size_t loom_hip_cache_decode_workspace_bytes(int64_t B, int64_t G, int64_t H, int64_t D, int64_t P,
                                             int64_t S, int weights) {
  if (B <= 0 || G <= 0 || H <= 0 || D <= 0 || P < 0 || S <= 0) return 0;
  if (P > (1 << 30) || S > (1 << 30) || !loom_prod_le({B, G, H, P + S, 4}, (int64_t)1 << 60))
    return SIZE_MAX;
  return align256((size_t)B * G * H * 8) + (size_t)B * G * H * (P + S) * 4;
}

int loom_hip_cache_decode(const void* prefix_k, const void* prefix_v, const void* k, const void* v,
                          const void* q, const void* lens, const void* weights, void* weights_out,
                          void* out, void* workspace, size_t workspace_bytes, int64_t B, int64_t G,
                          int64_t H, int64_t D, int64_t P, int64_t S, float scale, void* stream,
                          char* err, size_t errlen) {
  return cache_decode_impl<false>(prefix_k, prefix_v, k, v, q, lens, weights, weights_out, out,
                                  workspace, workspace_bytes, B, G, H, D, P, S, scale, stream, err,
                                  errlen);
}
int loom_hip_cache_decode_f16(const void* prefix_k, const void* prefix_v, const void* k,
                              const void* v, const void* q, const void* lens, const void* weights,
                              void* weights_out, void* out, void* workspace,
                              size_t workspace_bytes, int64_t B, int64_t G, int64_t H, int64_t D,
                              int64_t P, int64_t S, float scale, void* stream, char* err,
                              size_t errlen) {
  return cache_decode_impl<true>(prefix_k, prefix_v, k, v, q, lens, weights, weights_out, out,
                                 workspace, workspace_bytes, B, G, H, D, P, S, scale, stream, err,
                                 errlen);
}

}  // extern "C"
