// window.hip -- attention over a sliding window of each sequence's cache and its
// first tokens, on gfx950.  The reference has no counterpart: its @attention
// (attention.hip) sees every key, its @flash_decode (decode.hip) one length.
//
//   q, out [B, T, G, H, D]; k [B, G, D, S] (keys transposed), v [B, G, S, D];
//   lens [B], counts [B]: sequence b holds n = clamp(lens[b], 0, S) keys, of which
//   the last c = clamp(counts[b], 0, T) (all T without counts) are those of its
//   queries: row t < c is at position p = n - c + t and sees the keys
//     j <= p with j > p - window or j < sinks:
//   out = sum_j softmax_j(scale q . k_j) v_j.  A row that sees nothing is zero (p < 0
//   where a cache was cut since); rows t >= c are left as they are.
#include "common.h"

#include <cmath>

namespace {

struct WindowParams {
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  const int* lens;
  const int* counts;
  uint16_t* out;
  int B, G, H, D, T, S;
  int window, sinks;
  float c2;         // scale * log2(e)
};

// One wave to a row; 64 keys at a time, a lane to a key for the scores and to
// D / 64 columns for the values.
template <bool F16>
__global__ void __launch_bounds__(64) window_row_kernel(WindowParams p) {
  __shared__ float s_q[256], s_p[64];
  const int lane = threadIdx.x, GH = p.G * p.H;
  const int64_t row = blockIdx.x;
  const int gh = (int)(row % GH), g = gh / p.H;
  const int64_t bt = row / GH;
  const int b = (int)(bt / p.T), t = (int)(bt % p.T);
  const int n = min(max(p.lens[b], 0), p.S);
  const int c = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  if (t >= c) return;
  const int pos = n - c + t;
  const int lo = max(0, pos - p.window + 1);
  const uint16_t* k = p.k + ((int64_t)b * p.G + g) * p.D * p.S;
  const uint16_t* v = p.v + ((int64_t)b * p.G + g) * p.S * p.D;
  for (int d = lane; d < p.D; d += 64) s_q[d] = lo16<F16>(p.q[row * p.D + d]) * p.c2;
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  auto block = [&](int j0, int j1) {          // keys [j0, j1), at most 64
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < j1) {
      s = 0.f;
      for (int d = 0; d < p.D; ++d) s += s_q[d] * lo16<F16>(k[(int64_t)d * p.S + j]);
    }
    const float mb = fmaxf(m, wave_max(s));
    const float base = mb == -INFINITY ? 0.f : mb;
    const float e = j < j1 ? exp2f(s - base) : 0.f, r = exp2f(m - base);
    l = l * r + wave_sum(e);
    m = mb;
    s_p[lane] = e;
    __syncthreads();
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d >= p.D) break;
      float a = o[i] * r;
      for (int x = 0; x < j1 - j0; ++x) a += s_p[x] * lo16<F16>(v[(int64_t)(j0 + x) * p.D + d]);
      o[i] = a;
    }
    __syncthreads();
  };
  const int ns = min(min(p.sinks, lo), pos + 1);
  for (int j = 0; j < ns; j += 64) block(j, min(ns, j + 64));
  for (int j = lo; j <= pos; j += 64) block(j, min(pos + 1, j + 64));
  const float inv = l != 0.f ? 1.f / l : 0.f;
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < p.D) p.out[row * p.D + d] = (uint16_t)cvt16<F16>(o[i] * inv);
  }
}

template <bool F16>
int window_impl(const void* k, const void* v, const void* q, const void* lens, const void* counts,
                void* out, void* workspace, size_t workspace_bytes, int64_t B, int64_t G, int64_t H,
                int64_t D, int64_t T, int64_t S, int64_t window, int64_t sinks, float scale,
                void* stream, char* err, size_t errlen) {
  if (!k || !v || !q || !lens || !out)
    return loom_fail(err, errlen, LOOM_EINVAL, "window_attention: null tensor pointer");
  if (B <= 0 || G <= 0 || H <= 0 || D <= 0 || T <= 0 || S <= 0)
    return loom_fail(err, errlen, LOOM_EINVAL, "window_attention: extents must be positive");
  if (window < 1 || sinks < 0)
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "window_attention: window must be at least 1, sinks at least 0 (window=%lld "
                     "sinks=%lld)",
                     (long long)window, (long long)sinks);
  if (!(scale > 0.f) || !std::isfinite(scale))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "window_attention: scale must be finite and positive (got %g)", (double)scale);
  if (D % 8 != 0 || D > 256)
    return loom_fail(err, errlen, LOOM_EUNSUP,
                     "window_attention: head_dim %lld not built (a multiple of 8 up to 256)",
                     (long long)D);
  if (S > (1 << 29) || T > (1 << 29) || !loom_prod_le({B, G}, 65535) ||
      !loom_prod_le({T, H}, 1 << 29) || !loom_prod_le({B, G, cdiv64(T * H, 32)}, 1 << 23) ||
      !loom_prod_le({B, G, S, D}, (int64_t)1 << 50) ||
      !loom_prod_le({B, T, G, H, D}, (int64_t)1 << 50))
    return loom_fail(err, errlen, LOOM_EINVAL, "window_attention: problem too large");
  // a capacity that is not a multiple of 8 takes buffer descriptors, which address
  // one (b, g)'s keys in 32 bits
  if (S % 8 != 0 && !loom_prod_le({D, S, 2}, 0x7fffffffll))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "window_attention: D*S too large for an S that is not a multiple of 8");
  auto aligned = [](const void* p, uintptr_t n) {
    return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
  };
  if (!aligned(k, S % 8 == 0 ? 16 : 2) || !aligned16(v) || !aligned16(q) || !aligned16(out) ||
      !aligned(lens, 4) || !aligned(counts, 4))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "window_attention: tensors must be 16-byte aligned (k 2-byte when S is not a "
                     "multiple of 8; lens and counts 4-byte)");
  const size_t need = loom_hip_window_attention_workspace_bytes(B, G, H, D, T, S, window, sinks);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "window_attention: workspace needs %zu bytes (16-byte aligned), got %zu", need,
                     workspace_bytes);
  // out on q is safe: a workgroup reads its rows before it, or the join, writes them
  const int64_t cache = B * G * S * D * 2, rows = B * T * G * H * D * 2;
  const LoomSpan in[] = {{k, cache}, {v, cache}, {lens, B * 4}, {counts, B * 4},
                         {out == q ? nullptr : q, rows}},
                 outs[] = {{out, rows}, {need ? workspace : nullptr, (int64_t)need}};
  if (loom_outputs_overlap(in, outs))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "window_attention: out and the workspace must not overlap the other tensors or "
                     "each other (but out may be q)");
  WindowParams p{};
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q = static_cast<const uint16_t*>(q);
  p.lens = static_cast<const int*>(lens);
  p.counts = static_cast<const int*>(counts);
  p.out = static_cast<uint16_t*>(out);
  p.B = (int)B;
  p.G = (int)G;
  p.H = (int)H;
  p.D = (int)D;
  p.T = (int)T;
  p.S = (int)S;
  p.window = (int)std::min(window, S);
  p.sinks = (int)std::min(sinks, S);
  p.c2 = scale * 1.4426950408889634f;
  if (loom_validate_only()) return loom_ok(err, errlen);
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL((window_row_kernel<F16>), dim3((unsigned)(B * T * G * H)), dim3(64), 0, st, p);
  return loom_check_launch(err, errlen, "window_attention");
}

}  // namespace

extern "C" {

size_t loom_hip_window_attention_workspace_bytes(int64_t B, int64_t G, int64_t H, int64_t D,
                                                 int64_t T, int64_t S, int64_t window,
                                                 int64_t sinks) {
  return 0;
}

int loom_hip_window_attention(const void* k, const void* v, const void* q, const void* lens,
                              const void* counts, void* out, void* workspace,
                              size_t workspace_bytes, int64_t B, int64_t G, int64_t H, int64_t D,
                              int64_t T, int64_t S, int64_t window, int64_t sinks, float scale,
                              void* stream, char* err, size_t errlen) {
  return window_impl<false>(k, v, q, lens, counts, out, workspace, workspace_bytes, B, G, H, D, T,
                            S, window, sinks, scale, stream, err, errlen);
}
int loom_hip_window_attention_f16(const void* k, const void* v, const void* q, const void* lens,
                                  const void* counts, void* out, void* workspace,
                                  size_t workspace_bytes, int64_t B, int64_t G, int64_t H,
                                  int64_t D, int64_t T, int64_t S, int64_t window, int64_t sinks,
                                  float scale, void* stream, char* err, size_t errlen) {
  return window_impl<true>(k, v, q, lens, counts, out, workspace, workspace_bytes, B, G, H, D, T, S,
                           window, sinks, scale, stream, err, errlen);
}

}  // extern "C"
