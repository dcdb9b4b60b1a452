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

// Few tokens: a thread per element of one (token, sequence).
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

// Many tokens: a workgroup per 64 slots (a multiple of 64 first, so that whole
// 16-byte pieces of a K row are written) of one (b, g).  The tokens' K rows go
// to LDS as they are, DP elements apart, and come back transposed: a lane of
// ds_read_b64_tr_b16 gets four tokens of one d.  Each 32-lane pass reads 32
// bytes of rows k..k+3 and k+8..k+11; rows are whole 256-byte bank windows, so
// the XOR gives the eight rows distinct pairs of 16-byte chunks.
constexpr int kTok = 64;
LOOM_DEV int tok_swz(int k) { return 2 * ((k & 3) | ((k >> 1) & 4)); }

template <int DP>
__global__ void __launch_bounds__(256) cache_append_tile_kernel(AppendParams p) {
  __shared__ __attribute__((aligned(1024))) char smem[kTok * DP * 2];
  const int bg = blockIdx.y, b = bg / p.G, g = bg - b * p.G;
  const int n = cache_len(p.lens, b, p.S);
  const int c = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  const int tid = threadIdx.x;
  if (blockIdx.x == 0 && g == 0 && tid == 0) p.lens_out[b] = min(n + c, p.S);
  const int end = min(n + c, p.S);                     // slots n .. end-1 are written
  const int k0 = (n / kTok + (int)blockIdx.x) * kTok;  // this workgroup's slots
  if (k0 >= end) return;
  const int D = p.D, cpr = D / 8, S = p.S;             // 16-byte chunks of a row
  const int64_t row = (int64_t)p.G * D;                // elements from token to token
  // element 0 of slot k0's token (before the tensor for slots < n: not read)
  const int64_t src0 = ((int64_t)b * p.T + (k0 - n)) * row + (int64_t)g * D;
  uint16_t* const vo = p.v + ((int64_t)bg * S + k0) * D;
  for (int e = tid; e < kTok * cpr; e += 256) {
    const int k = e / cpr, ch = e - k * cpr;
    if (k0 + k < n || k0 + k >= end) continue;
    const int64_t src = src0 + k * row + ch * 8;
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p.nk + src);
    const u32x4_t y = *reinterpret_cast<const u32x4_t*>(p.nv + src);
    *reinterpret_cast<u32x4_t*>(smem + k * (DP * 2) + ((ch ^ tok_swz(k)) * 16)) = x;
    *reinterpret_cast<u32x4_t*>(vo + (int64_t)k * D + ch * 8) = y;
  }
  if (p.w && tid < kTok && k0 + tid >= n && k0 + tid < end) p.w[(int64_t)bg * S + k0 + tid] = 0.f;
  __syncthreads();
  // wave w: 16 rows d at a time; lane group q tokens 8 q .. 8 q + 7 of 32
  const int lane = tid & 63, wave = tid >> 6;
  const int r = lane & 15, q = lane >> 4, a4 = r >> 2, c4 = r & 3;
  const int64_t ko = (int64_t)bg * D * S;
  for (int x = wave; x < (D + 15) / 16 * 2; x += 4) {
    const int dt = x >> 1, kk = 32 * (x & 1) + 8 * q;  // first of this lane's eight slots
    const int ch = 2 * dt + (c4 >> 1);
    const lds_char_t* const base = (lds_char_t*)smem + (c4 & 1) * 8;
    const u32x2_t lo = lds_read_tr16(base + (kk + a4) * (DP * 2) + ((ch ^ tok_swz(kk + a4)) * 16));
    const u32x2_t hi =
        lds_read_tr16(base + (kk + 4 + a4) * (DP * 2) + ((ch ^ tok_swz(kk + 4 + a4)) * 16));
    const int d = 16 * dt + r, at = k0 + kk;
    if (d >= D) continue;
    uint16_t* const to = p.k + ko + (int64_t)d * S + at;
    const u32x4_t v = u32x4_t{lo[0], lo[1], hi[0], hi[1]};
    if (at >= n && at + 8 <= end) {
      __builtin_memcpy(to, &v, 16);     // 16-byte aligned when S is a multiple of 8
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i >= n && at + i < end) to[i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
    }
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
  int nk, njk, rows_k;  // K parts of a (b, g): njk stretches of slots x rows_k rows each
};

// A weight as a whole number of the same order: NaN below -inf, -0 as +0.
LOOM_DEV uint32_t weight_key(float w) {
  const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelWaves = 16, kSel = 64 * kSelWaves;
constexpr int kBins = 2048;     // 11 bits a digit: three digits of a 32-bit key

// The kept slots of one (sequence, KV head), ascending, by one workgroup: a
// radix selection of the weights' keys (11, 11 and 10 bits, highest first) finds
// the smallest key that stays and how many of its equals do; each wave then
// counts what stays of its stretch of slots and writes it behind the waves
// before it.  A wave owns a contiguous stretch; with KPT > 0 its keys stay in
// registers (KPT a lane, slots 64 apart), else (KPT 0, longer caches) every pass
// reads the weights again.
template <int KPT>
__global__ void __launch_bounds__(kSel) cache_select_kernel(EvictParams p) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t s_part[kSelWaves], s_digit, s_left;
  __shared__ int s_sel[kSelWaves], s_eq[kSelWaves];
  const int bg = blockIdx.x, b = bg / p.G;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = cache_len(p.lens, b, p.S);
  int* const idx = p.index + (int64_t)bg * p.keep;
  if (bg - b * p.G == 0 && tid == 0) p.lens_out[b] = min(n, p.keep);
  if (n <= p.keep) {
    for (int j = tid; j < p.keep; j += kSel) idx[j] = j < n ? j : -1;
    return;
  }
  const float* const w = p.w + (int64_t)bg * p.S;
  const int lo = p.sinks, hi = n - p.recent;   // the slots that are weighed
  const int per = KPT > 0 ? KPT : (n + kSel - 1) / kSel;   // keys of a lane
  const int i0 = wave * per * 64;              // this wave's slots: i0 + 64 u + lane
  uint32_t reg[KPT > 0 ? KPT : 1];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      const int i = i0 + u * 64 + lane;
      reg[u] = weight_key(w[min(i, n - 1)]);
    }
  }
  auto each = [&](auto f) {
    if constexpr (KPT > 0) {
#pragma unroll
      for (int u = 0; u < KPT; ++u) f(i0 + u * 64 + lane, reg[u]);
    } else {
      for (int u = 0; u < per && i0 + u * 64 < n; ++u) {
        const int i = i0 + u * 64 + lane;
        f(i, weight_key(w[min(i, n - 1)]));
      }
    }
  };
  uint32_t left = (uint32_t)(p.keep - p.sinks - p.recent);   // how many weighed ones stay
  const bool none = left == 0;
  uint32_t prefix = 0;
  for (int pass = 0; pass < 3 && !none; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t above = pass == 0 ? 0u : ~0u << (pass == 1 ? 21 : 10);   // digits found
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
    for (int i = tid; i < kBins; i += kSel) hist[i] = 0;
    __syncthreads();
    each([&](int i, uint32_t key) {
      const bool in = i >= lo && i < hi && (key & above) == prefix;
      const uint32_t dig = (key >> shift) & mask;
      const uint64_t m = __builtin_amdgcn_ballot_w64(in);
      if (m == 0) return;
      // lanes of one digit (a stretch of equal weights) count as one
      const uint32_t d0 = __builtin_amdgcn_readlane(dig, __builtin_ctzll(m));
      const uint64_t same = __builtin_amdgcn_ballot_w64(in && dig == d0);
      if (in && dig != d0) atomicAdd(&hist[dig], 1u);
      if (lane == 0) atomicAdd(&hist[d0], (uint32_t)__popcll(same));
    });
    __syncthreads();
    // the digit at which the count from the top reaches `left`: two bins a
    // thread, highest first
    const int bin = kBins - 1 - 2 * tid;
    const uint32_t h0 = hist[bin], h1 = hist[bin - 1];
    uint32_t inc = h0 + h1;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const uint32_t o = __shfl_up(inc, m);
      if (lane >= m) inc += o;
    }
    if (lane == 63) s_part[wave] = inc;
    __syncthreads();
    uint32_t before = inc - h0 - h1;            // keys of higher digits
    for (int x = 0; x < wave; ++x) before += s_part[x];
    if (before < left && before + h0 >= left) {
      s_digit = bin;
      s_left = left - before;
    } else if (before + h0 < left && before + h0 + h1 >= left) {
      s_digit = bin - 1;
      s_left = left - before - h0;
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
  }
  // stays: above the threshold, and the first `left` equal to it
  int sel = 0, eq = 0;
  each([&](int i, uint32_t key) {
    const bool in = i < n, must = in && (i < lo || i >= hi), free = in && !must && !none;
    sel += __popcll(__builtin_amdgcn_ballot_w64(must || (free && key > prefix)));
    eq += __popcll(__builtin_amdgcn_ballot_w64(free && key == prefix));
  });
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
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  each([&](int i, uint32_t key) {
    const bool in = i < n, must = in && (i < lo || i >= hi), free = in && !must && !none;
    const bool same = free && key == prefix;
    const uint64_t eqm = __builtin_amdgcn_ballot_w64(same);
    const bool stays = must || (free && key > prefix) ||
                       (same && eqs + __popcll(eqm & below) < (int)left);
    const uint64_t m = __builtin_amdgcn_ballot_w64(stays);
    if (stays) idx[at + __popcll(m & below)] = i;
    at += __popcll(m);
    eqs += __popcll(eqm);
  });
}

// The kept keys moved.  K parts take rows_k rows d of one (b, g) and 1024 kept
// slots: a lane an element, so a load touches the few lines that 64 kept slots
// span (eight elements a lane, for 16-byte stores, touched 64 of them); the
// slots stay in registers over the rows.  V parts take rows of D elements, 16
// bytes a lane, and the weights.
constexpr int kMoveK = 4;           // slots of a thread
constexpr int kMoveV = 64;          // slots of a V part
__global__ void __launch_bounds__(256) cache_move_kernel(EvictParams p) {
  const int bg = blockIdx.y, b = bg / p.G, tid = threadIdx.x;
  const int n = min(cache_len(p.lens, b, p.S), p.keep);
  const int* const idx = p.index + (int64_t)bg * p.keep;
  const int D = p.D;
  int x = blockIdx.x;
  if (x < p.nk) {
    const int j0 = x % p.njk * (256 * kMoveK) + tid, d0 = x / p.njk * p.rows_k;
    if (j0 - tid >= n) return;
    int at[kMoveK];
#pragma unroll
    for (int u = 0; u < kMoveK; ++u) at[u] = idx[min(j0 + 256 * u, n - 1)];
    const int d1 = min(D, d0 + p.rows_k);
    const uint16_t* src = p.k + ((int64_t)bg * D + d0) * p.S;
    uint16_t* dst = p.k_out + ((int64_t)bg * D + d0) * p.So;
#pragma unroll 4
    for (int d = d0; d < d1; ++d) {
      uint16_t e[kMoveK];
#pragma unroll
      for (int u = 0; u < kMoveK; ++u) e[u] = src[at[u]];
#pragma unroll
      for (int u = 0; u < kMoveK; ++u)
        if (j0 + 256 * u < n) dst[j0 + 256 * u] = e[u];
      src += p.S;
      dst += p.So;
    }
    return;
  }
  x -= p.nk;
  const int j0 = x * kMoveV, jn = min(kMoveV, n - j0);
  if (jn <= 0) return;
  if (tid < jn) p.w_out[(int64_t)bg * p.So + j0 + tid] = p.w[(int64_t)bg * p.S + idx[j0 + tid]];
  const int cpr = D / 8;
  const uint16_t* const src = p.v + (int64_t)bg * p.S * D;
  uint16_t* const dst = p.v_out + ((int64_t)bg * p.So + j0) * D;
#pragma unroll 4
  for (int e = tid; e < jn * cpr; e += 256) {
    const int j = e / cpr, c = e - j * cpr;
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(src + (int64_t)idx[j0 + j] * D + c * 8);
    *reinterpret_cast<u32x4_t*>(dst + (int64_t)j * D + c * 8) = v;
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
  if (S > (1 << 29) || T > (1 << 29) || !loom_prod_le({B, G}, 65535) ||
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
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (T < 16) {
    hipLaunchKernelGGL(cache_append_kernel, dim3((unsigned)T, (unsigned)B), dim3(256), 0, st, p);
  } else {
    // slots that a sequence's tokens reach from any length: T and the part of a
    // tile before them
    const dim3 grid((unsigned)(cdiv64(std::min(T, S), kTok) + 1), (unsigned)(B * G));
    if (D <= 128)
      hipLaunchKernelGGL(cache_append_tile_kernel<128>, grid, dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL(cache_append_tile_kernel<256>, grid, dim3(256), 0, st, p);
  }
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
  if (S > (1 << 29) || S_out > (1 << 29) || !loom_prod_le({B, G}, 65535) ||
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
  const dim3 sel((unsigned)(B * G)), selb(kSel);
  if (S <= 4 * kSel) hipLaunchKernelGGL(cache_select_kernel<4>, sel, selb, 0, st, p);
  else if (S <= 16 * kSel) hipLaunchKernelGGL(cache_select_kernel<16>, sel, selb, 0, st, p);
  else hipLaunchKernelGGL(cache_select_kernel<0>, sel, selb, 0, st, p);
  int rc = loom_check_launch(err, errlen, "cache_evict (select)");
  if (rc) return rc;
  // rows of a K part: as many (up to 16) as leave about 1024 parts
  p.njk = (int)cdiv64(keep, 256 * kMoveK);
  p.rows_k = (int)std::max<int64_t>(2, std::min<int64_t>(16, B * G * p.njk * D / 1024));
  p.nk = (int)(p.njk * cdiv64(D, p.rows_k));
  const dim3 grid((unsigned)(p.nk + cdiv64(keep, kMoveV)), (unsigned)(B * G));
  hipLaunchKernelGGL(cache_move_kernel, grid, dim3(256), 0, st, p);
  return loom_check_launch(err, errlen, "cache_evict (move)");
}

}  // extern "C"
