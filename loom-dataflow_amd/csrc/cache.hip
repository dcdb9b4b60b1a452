// cache.hip -- a serving loop's caches of different lengths on gfx950: new
// tokens appended (cache_append) and each cache cut to its heaviest keys
// (cache_evict).  cache_decode.hip has the attention that reads them.  The
// reference has no counterpart of these.
//
//   k [B, G, D, S] (keys transposed), v [B, G, S, D], lens [B] int32: sequence
//   b holds n = clamp(lens[b], 0, S) keys in slots 0 .. n-1 of each of its G
//   KV heads; what the slots behind them hold is never used.
//   append: k[b, g, :, n + t] = new_k[b, t, g, :], v[b, g, n + t, :] =
//           new_v[b, t, g, :] for t < counts[b] (slots past S are dropped), and
//           their weights zero.
//   evict:  of n > keep keys the first `sinks`, the last `recent` and, of the
//           others, the keep - sinks - recent of largest weight stay (ties:
//           the lowest slot; NaN below everything), in the order of their
//           slots.
#include "common.h"

namespace {

LOOM_DEV int cache_len(const int* lens, int b, int S) { return min(max(lens[b], 0), S); }

struct AppendParams {
  uint16_t* k;
  uint16_t* v;
  float* w;            // null: none
  const uint16_t* nk;
  const uint16_t* nv;
  const int* lens;
  const int* counts;   // null: T each
  int* lens_out;
  int B, G, D, S, T;
};

// One workgroup per (new token, sequence): a thread per (g, d) element.
__global__ void __launch_bounds__(256) cache_append_kernel(AppendParams p) {
  const int t = blockIdx.x, b = blockIdx.y;
  const int n = cache_len(p.lens, b, p.S);
  const int c = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  if (t == 0 && threadIdx.x == 0) p.lens_out[b] = min(n + c, p.S);
  const int at = n + t;
  if (t >= c || at >= p.S) return;
  for (int e = threadIdx.x; e < p.G * p.D; e += 256) {
    const int g = e / p.D, d = e % p.D;
    const int64_t src = ((int64_t)b * p.T + t) * p.G * p.D + e;
    const int64_t bg = (int64_t)b * p.G + g;
    p.k[(bg * p.D + d) * p.S + at] = p.nk[src];
    p.v[(bg * p.S + at) * p.D + d] = p.nv[src];
    if (p.w && d == 0) p.w[bg * p.S + at] = 0.f;
  }
}

struct EvictParams {
  const uint16_t* k;
  const uint16_t* v;
  const float* w;
  const int* lens;
  uint16_t* k_out;
  uint16_t* v_out;
  float* w_out;
  int* lens_out;
  int* index;          // [B, G, keep]
  int B, G, D, S, So, keep, recent, sinks;
};

// A weight as a whole number of the same order: NaN below -inf, -0 as +0.
LOOM_DEV uint32_t weight_key(float w) {
  const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelWaves = 16;

// The kept slots of one (sequence, KV head), ascending, by one workgroup: a
// radix selection of the weights' keys (four digits of 8 bits, highest first)
// finds the smallest key that stays and how many of its equals do; each wave
// then counts what stays of its stretch of slots and writes it behind the
// waves before it.
__global__ void __launch_bounds__(64 * kSelWaves) cache_select_kernel(EvictParams p) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t s_digit, s_left;
  __shared__ int s_sel[kSelWaves], s_eq[kSelWaves];
  const int bg = blockIdx.x, b = bg / p.G;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = cache_len(p.lens, b, p.S);
  int* const idx = p.index + (int64_t)bg * p.keep;
  if (bg % p.G == 0 && tid == 0) p.lens_out[b] = min(n, p.keep);
  if (n <= p.keep) {
    for (int j = tid; j < p.keep; j += 64 * kSelWaves) idx[j] = j < n ? j : -1;
    return;
  }
  const float* const w = p.w + (int64_t)bg * p.S;
  const int lo = p.sinks, hi = n - p.recent;   // the slots that are weighed
  uint32_t left = (uint32_t)(p.keep - p.sinks - p.recent);   // how many of them stay
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0 && left > 0; shift -= 8) {
    for (int i = tid; i < 256; i += 64 * kSelWaves) hist[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += 64 * kSelWaves) {
      const uint32_t key = weight_key(w[i]);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t above = 0;
      int d = 255;
      while (d > 0 && above + hist[d] < left) above += hist[d--];
      s_digit = (uint32_t)d;
      s_left = left - above;
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
    __syncthreads();
  }
  // stays: above the threshold, and the first `left` equal to it
  const bool none = p.keep == p.sinks + p.recent;
  const int seg = (n + 64 * kSelWaves - 1) / (64 * kSelWaves) * 64;
  const int i0 = min(wave * seg, n), i1 = min(i0 + seg, n);
  int sel = 0, eq = 0;
  for (int i = i0 + lane; i < i1; i += 64) {
    const bool must = i < lo || i >= hi;
    const uint32_t key = must || none ? 0u : weight_key(w[i]);
    sel += must || (!none && key > prefix);
    eq += !must && !none && key == prefix;
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    sel += __shfl_xor(sel, m);
    eq += __shfl_xor(eq, m);
  }
  if (lane == 0) {
    s_sel[wave] = sel;
    s_eq[wave] = eq;
  }
  __syncthreads();
  int at = 0, eqs = 0;         // kept slots and threshold equals before this wave
  for (int x = 0; x < wave; ++x) {
    at += s_sel[x];
    eqs += s_eq[x];
  }
  at += min(eqs, (int)left);
  for (int base = i0; base < i1; base += 64) {
    const int i = base + lane;
    const bool in = i < i1, must = in && (i < lo || i >= hi);
    const uint32_t key = !in || must || none ? 0u : weight_key(w[i]);
    const bool same = in && !must && !none && key == prefix;
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    const uint64_t eqm = __builtin_amdgcn_ballot_w64(same);
    const bool stays = must || (in && !none && key > prefix) ||
                       (same && eqs + __popcll(eqm & below) < (int)left);
    const uint64_t m = __builtin_amdgcn_ballot_w64(stays);
    if (stays) idx[at + __popcll(m & below)] = i;
    at += __popcll(m);
    eqs += __popcll(eqm);
  }
}

// Rows of the kept slots: K elements of row d (blockIdx.y < D), V and weights.
__global__ void __launch_bounds__(256) cache_gather_kernel(EvictParams p) {
  const int bg = blockIdx.z, y = blockIdx.y;
  const int n = min(cache_len(p.lens, bg / p.G, p.S), p.keep);
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= n) return;
  const int i = p.index[(int64_t)bg * p.keep + j];
  if (y < p.D) {
    p.k_out[((int64_t)bg * p.D + y) * p.So + j] = p.k[((int64_t)bg * p.D + y) * p.S + i];
    p.v_out[((int64_t)bg * p.So + j) * p.D + y] = p.v[((int64_t)bg * p.S + i) * p.D + y];
  } else {
    p.w_out[(int64_t)bg * p.So + j] = p.w[(int64_t)bg * p.S + i];
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Whether [a, a + an) and [b, b + bn) share a byte.
bool overlap(const void* a, int64_t an, const void* b, int64_t bn) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + (uint64_t)bn && y < x + (uint64_t)an;
}

}  // namespace

extern "C" {

int loom_hip_cache_append(void* k, void* v, void* weights, const void* lens, const void* new_k,
                          const void* new_v, const void* counts, void* lens_out, int64_t B,
                          int64_t G, int64_t D, int64_t S, int64_t T, void* stream, char* err,
                          size_t errlen) {
  if (!k || !v || !lens || !new_k || !new_v || !lens_out)
    return loom_fail(err, errlen, LOOM_EINVAL, "cache_append: null tensor pointer");
  if (B <= 0 || G <= 0 || D <= 0 || S <= 0 || T <= 0)
    return loom_fail(err, errlen, LOOM_EINVAL, "cache_append: extents must be positive");
  if (D % 8 != 0 || D > 256)
    return loom_fail(err, errlen, LOOM_EUNSUP,
                     "cache_append: head_dim %lld not built (a multiple of 8 up to 256)",
                     (long long)D);
  if (S > (1 << 30) || T > (1 << 30) || !loom_prod_le({B, G}, 65535) ||
      !loom_prod_le({B, G, S, D}, (int64_t)1 << 50) ||
      !loom_prod_le({B, G, T, D}, (int64_t)1 << 50))
    return loom_fail(err, errlen, LOOM_EINVAL, "cache_append: problem too large");
  if (!aligned(k, S % 8 == 0 ? 16 : 2) || !aligned(v, 16) || !aligned(new_k, 16) ||
      !aligned(new_v, 16) || !aligned(weights, 4) || !aligned(lens, 4) || !aligned(counts, 4) ||
      !aligned(lens_out, 4))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_append: v, new_k and new_v must be 16-byte aligned, k 16-byte (2-byte "
                     "when S is not a multiple of 8), the others 4-byte");
  if (overlap(lens, 4 * B, lens_out, 4 * B) || (counts && overlap(counts, 4 * B, lens_out, 4 * B)))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_append: lens_out must not overlap lens or counts");
  AppendParams p{};
  p.k = static_cast<uint16_t*>(k);
  p.v = static_cast<uint16_t*>(v);
  p.w = static_cast<float*>(weights);
  p.nk = static_cast<const uint16_t*>(new_k);
  p.nv = static_cast<const uint16_t*>(new_v);
  p.lens = static_cast<const int*>(lens);
  p.counts = static_cast<const int*>(counts);
  p.lens_out = static_cast<int*>(lens_out);
  p.B = (int)B;
  p.G = (int)G;
  p.D = (int)D;
  p.S = (int)S;
  p.T = (int)T;
  if (loom_validate_only()) return loom_ok(err, errlen);
  hipLaunchKernelGGL(cache_append_kernel, dim3((unsigned)T, (unsigned)B), dim3(256), 0,
                     static_cast<hipStream_t>(stream), p);
  return loom_check_launch(err, errlen, "cache_append");
}

int loom_hip_cache_evict(const void* k, const void* v, const void* weights, const void* lens,
                         void* k_out, void* v_out, void* weights_out, void* lens_out, void* index,
                         int64_t B, int64_t G, int64_t D, int64_t S, int64_t S_out, int64_t keep,
                         int64_t recent, int64_t sinks, void* stream, char* err, size_t errlen) {
  if (!k || !v || !weights || !lens || !k_out || !v_out || !weights_out || !lens_out || !index)
    return loom_fail(err, errlen, LOOM_EINVAL, "cache_evict: null tensor pointer");
  if (B <= 0 || G <= 0 || D <= 0 || S <= 0 || S_out <= 0)
    return loom_fail(err, errlen, LOOM_EINVAL, "cache_evict: extents must be positive");
  if (keep <= 0 || keep > S_out || recent < 0 || sinks < 0 || recent > keep || sinks > keep - recent)
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_evict: must satisfy 1 <= keep <= S_out, 0 <= recent, sinks and "
                     "recent + sinks <= keep (keep=%lld recent=%lld sinks=%lld S_out=%lld)",
                     (long long)keep, (long long)recent, (long long)sinks, (long long)S_out);
  if (D % 8 != 0 || D > 256)
    return loom_fail(err, errlen, LOOM_EUNSUP,
                     "cache_evict: head_dim %lld not built (a multiple of 8 up to 256)",
                     (long long)D);
  if (S > (1 << 30) || S_out > (1 << 30) || !loom_prod_le({B, G}, 65535) ||
      !loom_prod_le({B, G, S, D}, (int64_t)1 << 50) ||
      !loom_prod_le({B, G, S_out, D}, (int64_t)1 << 50))
    return loom_fail(err, errlen, LOOM_EINVAL, "cache_evict: problem too large");
  if (!aligned(k, S % 8 == 0 ? 16 : 2) || !aligned(v, 16) ||
      !aligned(k_out, S_out % 8 == 0 ? 16 : 2) || !aligned(v_out, 16) || !aligned(weights, 4) ||
      !aligned(weights_out, 4) || !aligned(lens, 4) || !aligned(lens_out, 4) || !aligned(index, 4))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_evict: v and v_out must be 16-byte aligned, k and k_out 16-byte (2-byte "
                     "when their capacity is not a multiple of 8)");
  const int64_t kin = B * G * S * D * 2, kout = B * G * S_out * D * 2;
  const struct { const void* p; int64_t n; } in[4] = {
      {k, kin}, {v, kin}, {weights, B * G * S * 4}, {lens, B * 4}},
      out[5] = {{k_out, kout}, {v_out, kout}, {weights_out, B * G * S_out * 4}, {lens_out, B * 4},
                {index, B * G * keep * 4}};
  for (const auto& o : out) {
    bool bad = false;
    for (const auto& i : in) bad |= overlap(i.p, i.n, o.p, o.n);
    for (const auto& x : out) bad |= &x != &o && overlap(x.p, x.n, o.p, o.n);
    if (bad)
      return loom_fail(err, errlen, LOOM_EINVAL,
                       "cache_evict: outputs must not overlap the inputs or each other");
  }
  EvictParams p{};
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.w = static_cast<const float*>(weights);
  p.lens = static_cast<const int*>(lens);
  p.k_out = static_cast<uint16_t*>(k_out);
  p.v_out = static_cast<uint16_t*>(v_out);
  p.w_out = static_cast<float*>(weights_out);
  p.lens_out = static_cast<int*>(lens_out);
  p.index = static_cast<int*>(index);
  p.B = (int)B;
  p.G = (int)G;
  p.D = (int)D;
  p.S = (int)S;
  p.So = (int)S_out;
  p.keep = (int)keep;
  p.recent = (int)recent;
  p.sinks = (int)sinks;
  if (loom_validate_only()) return loom_ok(err, errlen);
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(cache_select_kernel, dim3((unsigned)(B * G)), dim3(64 * kSelWaves), 0, st, p);
  int rc = loom_check_launch(err, errlen, "cache_evict (select)");
  if (rc) return rc;
  const dim3 grid((unsigned)cdiv64(keep, 256), (unsigned)D + 1, (unsigned)(B * G));
  hipLaunchKernelGGL(cache_gather_kernel, grid, dim3(256), 0, st, p);
  return loom_check_launch(err, errlen, "cache_evict (gather)");
}

}  // extern "C"
