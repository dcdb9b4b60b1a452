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

#include <type_traits>

namespace {

LOOM_DEV int cache_len(const int* lens, int b, int S) { return min(max(lens[b], 0), S); }

// 16 bytes to any element of a row, non-temporal (as store_stream: the written
// rows, which nothing here reads back, displace no rows still to be read and are
// not left to the flush at the kernel's end: evictions of B8 G8 D64 S16383 93 ->
// 79 us, B32 S8192 33 -> 29; appended prompts 39.4 -> 36.7)
typedef u32x4_t any16_t __attribute__((aligned(2)));
LOOM_DEV void store_any16(uint16_t* to, const u32x4_t& v) {
  __builtin_nontemporal_store(v, reinterpret_cast<any16_t*>(to));
}

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

// Few tokens: a thread per element of one (token, sequence).  A token's K
// elements lie S apart, a line of the cache each: latency bounds it (B32 G1 D128:
// 2.4 us).
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
// the XOR gives the eight rows distinct pairs of 16-byte chunks.  Bound by memory:
// B8 G8 D128, prompts of 1024 to 4096 tokens (180 MB read and written) 38 us, 4.7
// TB/s.
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
    store_stream(reinterpret_cast<u32x4_t*>(vo + (int64_t)k * D + ch * 8), y);
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
      store_any16(to, v);               // 16-byte aligned when S is a multiple of 8
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
  int slots_v;          // slots of a V part, at most 256
};

// A weight as a whole number of the same order, above 0: NaN below -inf (1), -0
// as +0 (what the addition gives).
LOOM_DEV uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return w == w ? k : 1u;
}

constexpr int kSelWaves = 16, kSel = 64 * kSelWaves;
constexpr int kBins = 4096;     // 12 bits of the first digit, 10 of the others
// copies of the histogram (lane l counts in copy l % 4: fewer lanes of one
// instruction meet in a bin), 16 banks apart
constexpr int kCopies = 4, kCopyStep = kBins + 16;
constexpr int kList = 256;

LOOM_DEV int lanes_below(uint64_t m) {   // set lanes below this one
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32),
                                        __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
}
// Inclusive sum over the lanes below: DPP adds (a shuffle goes through the LDS
// unit, which sixteen waves share here).
template <int CTRL, int ROWS>
LOOM_DEV uint32_t dpp_add(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
LOOM_DEV uint32_t row_scan(uint32_t v) {   // within 16 lanes
  v = dpp_add<0x111, 0xf>(v);              // row_shr:1, 2, 4, 8
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  return dpp_add<0x118, 0xf>(v);
}
LOOM_DEV uint32_t lane_scan(uint32_t v) {
  v = row_scan(v);
  v = dpp_add<0x142, 0xa>(v);              // row_bcast:15 into rows 1 and 3
  return dpp_add<0x143, 0xc>(v);           // row_bcast:31 into rows 2 and 3
}
// Sum of the 16 waves' values below `wave`.
LOOM_DEV uint32_t waves_before(const uint32_t* v, int lane, int wave) {
  const uint32_t x = row_scan(lane < wave ? v[lane & (kSelWaves - 1)] : 0u);
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 15);
}

// The kept slots of one (sequence, KV head), ascending, by one workgroup: a
// histogram of the weights' keys by their first 12 bits (sign, exponent, 3 bits)
// finds the bin with the smallest key that stays; if it holds at most 256 keys,
// one wave finds that key among them bit by bit, else two more digits of 10 bits
// are counted.  Each wave then counts what stays of its stretch of slots and
// writes it behind the waves before it.  Sinks and recent slots take the highest
// key and slots behind the length 0, below every weight's, so no pass looks at
// slot numbers: the instructions per key bound this kernel (a CU's four SIMDs
// each run four of its waves).  With KPT > 0 the keys stay in registers (KPT a
// lane, slots 64 apart; in LDS, with rolled loops, 23 us against 15 at 16 a
// lane), else (KPT 0, longer caches) every pass reads the weights again,
// eight a lane at a time (8 x 70000: 57 us against 88 one by one).  4096 weights
// 6.0 us, 32 x 8192 8.6 us, 64 x 16383 11.8 us, 8 x 32768 19.0 us.
template <int KPT>
__global__ void __launch_bounds__(kSel) cache_select_kernel(EvictParams p) {
  __shared__ __attribute__((aligned(16))) uint32_t hist[kCopyStep * kCopies], s_list[kList];
  __shared__ uint32_t s_part[kSelWaves], s_digit, s_left, s_count, s_n;
  __shared__ uint32_t s_sel[kSelWaves], s_eq[kSelWaves];
  const int bg = blockIdx.x, b = bg / p.G;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the weights are on their way with the length
  const rsrc_t w = make_rsrc(p.w + (int64_t)bg * p.S, (uint32_t)p.S * 4u);
  auto load = [&](int i) { return __uint_as_float(buf_load4(w, (uint32_t)i * 4u)); };
  float x[KPT > 0 ? KPT : 1];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int u = 0; u < KPT; ++u) x[u] = load((wave * KPT + u) * 64 + lane);
  }
  const int n = cache_len(p.lens, b, p.S);
  auto clear = [&]() {
    for (int i = tid; i < kCopyStep * kCopies / 4; i += kSel)
      *reinterpret_cast<u32x4_t*>(hist + 4 * i) = u32x4_t{0u, 0u, 0u, 0u};
  };
  clear();
  if (tid == 0) s_n = 0;
  int* const idx = p.index + (int64_t)bg * p.keep;
  if (bg - b * p.G == 0 && tid == 0) p.lens_out[b] = min(n, p.keep);
  if (n <= p.keep) {
    for (int j = tid; j < p.keep; j += kSel) idx[j] = j < n ? j : -1;
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;   // the slots that are weighed
  const int per = KPT > 0 ? KPT : (n + kSel - 1) / kSel;   // keys of a lane
  const int i0 = wave * per * 64;              // this wave's slots: i0 + 64 u + lane
  auto key_of = [&](int base, float v) {       // of slot base + lane
    uint32_t k = weight_key(v);
    if (base < lo || base + 64 > hi) {         // wave-uniform
      const int i = base + lane;
      k = i < lo || i >= hi ? (i < n ? ~0u : 0u) : k;
    }
    return k;
  };
  uint32_t reg[KPT > 0 ? KPT : 1];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int u = 0; u < KPT; ++u) reg[u] = key_of(i0 + u * 64, x[u]);
  }
  auto each = [&](auto f) {                    // f(first slot of the wave's 64, key)
    if constexpr (KPT > 0) {
#pragma unroll
      for (int u = 0; u < KPT; ++u) f(i0 + u * 64, reg[u]);
    } else {
      for (int u0 = 0; u0 < per && i0 + u0 * 64 < n; u0 += 8) {
        float y[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) y[u] = load(i0 + (u0 + u) * 64 + lane);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (u0 + u < per) f(i0 + (u0 + u) * 64, key_of(i0 + (u0 + u) * 64, y[u]));
      }
    }
  };
  uint32_t left = (uint32_t)p.keep;            // how many stay; n > keep keys are above 0
  uint32_t prefix = 0, found = 0;              // the threshold's digits and their mask
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = 20 - 10 * pass;
    const uint32_t mask = pass == 0 ? kBins - 1 : 1023u;
    if (pass > 0) clear();
    __syncthreads();
    uint32_t* const mine = hist + lane % kCopies * kCopyStep;
    if (pass == 0)
      each([&](int, uint32_t key) {
        if (key != 0u) atomicAdd(&mine[key >> 20], 1u);
      });
    else
      each([&](int, uint32_t key) {
        if (key != 0u && (key & found) == prefix) atomicAdd(&mine[(key >> shift) & mask], 1u);
      });
    __syncthreads();
    // the digit at which the count from the top reaches `left`: four bins a
    // thread, highest first
    const int bin = kBins - 4 - 4 * tid;
    u32x4_t h = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
    for (int c = 0; c < kCopies; ++c)
      h += *reinterpret_cast<const u32x4_t*>(hist + c * kCopyStep + bin);
    const uint32_t sum = h[0] + h[1] + h[2] + h[3];
    const uint32_t inc = lane_scan(sum);
    if (lane == 63) s_part[wave] = inc;
    __syncthreads();
    uint32_t before = inc - sum + waves_before(s_part, lane, wave);   // keys of higher digits
    if (before < left && before + sum >= left) {
      int d = 3;
#pragma unroll
      for (int c = 3; c > 0; --c)
        if (d == c && before + h[c] < left) {
          before += h[c];
          d = c - 1;
        }
      s_digit = bin + d;
      s_left = left - before;
      s_count = d == 3 ? h[3] : d == 2 ? h[2] : d == 1 ? h[1] : h[0];
    }
    __syncthreads();
    prefix |= s_digit << shift;
    found |= mask << shift;
    left = s_left;
    const int cnt = (int)s_count;
    if (pass == 2 || cnt > kList) continue;
    // few enough: into a list, each lane's behind those of the lanes before it
    int c = 0;
    each([&](int, uint32_t key) { c += key != 0u && (key & found) == prefix; });
    if (__builtin_amdgcn_ballot_w64(c != 0) != 0) {
      int to = (int)lane_scan((uint32_t)c);
      const int all = __builtin_amdgcn_readlane(to, 63);
      uint32_t at = 0;
      if (lane == 0) at = atomicAdd(&s_n, (uint32_t)all);
      to += (int)__builtin_amdgcn_readfirstlane(at) - c;
      each([&](int, uint32_t key) {
        if (key != 0u && (key & found) == prefix) s_list[to++] = key;
      });
    }
    __syncthreads();
    if (wave == 0) {                           // the left-th largest of the list
      uint32_t k[kList / 64], t = prefix;
#pragma unroll
      for (int y = 0; y < kList / 64; ++y) k[y] = 64 * y + lane < cnt ? s_list[64 * y + lane] : 0u;
      auto above = [&](uint32_t v) {
        uint32_t m = 0;
#pragma unroll
        for (int y = 0; y < kList / 64; ++y) m += __popcll(__builtin_amdgcn_ballot_w64(k[y] > v));
        return m;
      };
      for (uint32_t bit = 1u << (shift - 1); bit != 0; bit >>= 1)
        if (above((t | bit) - 1) >= left) t |= bit;
      const uint32_t gt = above(t);
      if (lane == 0) {
        s_digit = t;
        s_left = left - gt;
      }
    }
    __syncthreads();
    prefix = s_digit;
    left = s_left;
    break;
  }
  // stays: above the threshold, and the first `left` equal to it
  int sel = 0, eq = 0;
  each([&](int, uint32_t key) {
    sel += __popcll(__builtin_amdgcn_ballot_w64(key > prefix));
    eq += __popcll(__builtin_amdgcn_ballot_w64(key == prefix));
  });
  if (lane == 0) {
    s_sel[wave] = sel;
    s_eq[wave] = eq;
  }
  __syncthreads();
  // kept slots and threshold equals before this wave
  int eqs = (int)waves_before(s_eq, lane, wave);
  int at = (int)waves_before(s_sel, lane, wave) + min(eqs, (int)left);
  each([&](int i, uint32_t key) {
    uint64_t m = __builtin_amdgcn_ballot_w64(key > prefix);
    const uint64_t eqm = __builtin_amdgcn_ballot_w64(key == prefix);
    if (eqm != 0) {
      m |= __builtin_amdgcn_ballot_w64(key == prefix && eqs + lanes_below(eqm) < (int)left);
      eqs += __popcll(eqm);
    }
    if ((m >> lane) & 1) idx[at + lanes_below(m)] = i + lane;
    at += __popcll(m);
  });
}

// The kept keys moved.  A wave of a K part takes 512 kept slots, eight
// consecutive ones a lane, over rows_k rows d: the stretch of the source row that
// they span comes in 16-byte pieces, goes through LDS and leaves as 16-byte
// pieces of the packed row (a 2-byte load and store per element moved the same
// rows at 2.7 TB/s, bound by the address unit).  A stretch longer than a window of
// 4096 slots goes through it piece by piece.  V parts take slots_v rows of D
// elements, 16 bytes a lane, and the weights.
constexpr int kMoveJ = 512, kMoveWin = 4096, kMoveP = kMoveWin / 512;

// eight elements of a row from slot i on (zeros past n)
LOOM_DEV u32x4_t row_slots8(const uint16_t* row, int i, int n) {
  u32x4_t v = u32x4_t{0u, 0u, 0u, 0u};
  if (i + 8 <= n) {
    __builtin_memcpy(&v, row + i, 16);
  } else {
#pragma unroll 1
    for (int e = 0; e < 8 && i + e < n; ++e) {
      const uint32_t h = (uint32_t)row[i + e] << (16 * (e & 1));
      v[0] |= e / 2 == 0 ? h : 0u;
      v[1] |= e / 2 == 1 ? h : 0u;
      v[2] |= e / 2 == 2 ? h : 0u;
      v[3] |= e / 2 == 3 ? h : 0u;
    }
  }
  return v;
}

// eight kept elements of a row, slots j .. j + 7 of n
LOOM_DEV void store_slots8(uint16_t* to, const uint32_t (&h)[8], int j, int n) {
  if (j + 8 <= n) {
    store_any16(to, u32x4_t{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16,
                            h[6] | h[7] << 16});
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (j + e < n) to[e] = (uint16_t)h[e];
  }
}

// The rows of kept slots that span one window, NP pieces of 512 slots to a row, 8 / NP
// rows at a time: eight 16-byte loads a lane are in flight whatever stretch the kept
// slots span.
template <int NP>
LOOM_DEV void move_rows(const EvictParams& p, const uint16_t* src, uint16_t* dst, int rows,
                        const int (&at)[8], int s0, int len, int j, int n, int lane,
                        uint16_t* win) {
  constexpr int RB = kMoveP / NP;
  u32x4_t piece[RB][NP];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      if (r0 + rb < rows)
#pragma unroll
        for (int u = 0; u < NP; ++u)
          if (u * 512 < len)
            piece[rb][u] = row_slots8(src + (int64_t)(r0 + rb) * p.S, s0 + u * 512 + 8 * lane, p.S);
  };
  fetch(0);
  for (int r0 = 0; r0 < rows; r0 += RB) {
    lds_order();
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      if (r0 + rb < rows)
#pragma unroll
        for (int u = 0; u < NP; ++u)
          if (u * 512 < len)
            *reinterpret_cast<u32x4_t*>(win + (rb * NP + u) * 512 + 8 * lane) = piece[rb][u];
    lds_order();
    fetch(r0 + RB);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      if (r0 + rb < rows) {
        const uint16_t* from = win + rb * NP * 512;
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = from[at[e] - s0];
        store_slots8(dst + (int64_t)(r0 + rb) * p.So, h, j, n);
      }
  }
}

// The rows of kept slots that lie further apart: window after window of a row, each
// lane picking up what it has there, one store when the row is through (stores of
// what each window held, 2 bytes each: B8 G8 S16383 -> 1024 95.9 us a call against
// 66.5).
LOOM_DEV void move_far(const EvictParams& p, const uint16_t* src, uint16_t* dst, int rows,
                       const int (&at)[8], int s0, int last, int j, int n, int lane,
                       uint16_t* win) {
  u32x4_t piece[kMoveP];
  auto fetch = [&](int row, int w0) {
#pragma unroll
    for (int u = 0; u < kMoveP; ++u)
      if (u * 512 <= last - w0)
        piece[u] = row_slots8(src + (int64_t)row * p.S, w0 + u * 512 + 8 * lane, p.S);
  };
  uint32_t h[8] = {};
  fetch(0, s0);
  for (int row = 0, w0 = s0; row < rows;) {
    lds_order();
#pragma unroll
    for (int u = 0; u < kMoveP; ++u)
      if (u * 512 <= last - w0)
        *reinterpret_cast<u32x4_t*>(win + u * 512 + 8 * lane) = piece[u];
    lds_order();
    const bool end = last - w0 < kMoveWin;
    const int row1 = row + end, w1 = end ? s0 : w0 + kMoveWin;
    if (row1 < rows) fetch(row1, w1);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // clamped: lanes without a slot here read the same two places
      const uint32_t x = win[min(max(at[e] - w0, 0), kMoveWin - 1)];
      h[e] = (uint32_t)(at[e] - w0) < (uint32_t)kMoveWin ? x : h[e];
    }
    if (end) store_slots8(dst + (int64_t)row * p.So, h, j, n);
    row = row1;
    w0 = w1;
  }
}

__global__ void __launch_bounds__(256) cache_move_kernel(EvictParams p) {
  __shared__ __attribute__((aligned(16))) uint16_t s_win[4][kMoveWin];
  const int bg = blockIdx.y, b = bg / p.G, tid = threadIdx.x;
  const int n = min(cache_len(p.lens, b, p.S), p.keep);
  const int* const idx = p.index + (int64_t)bg * p.keep;
  const int D = p.D;
  int x = blockIdx.x;
  if (x < p.nk) {
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int jc = x % p.njk * kMoveJ;
    const int d0 = (x / p.njk * 4 + wave) * p.rows_k, rows = min(D - d0, p.rows_k);
    if (jc >= n || rows <= 0) return;
    const int j = jc + 8 * lane;                // this lane's kept slots j .. j + 7
    int at[8];
    if (j + 8 <= n) {
      __builtin_memcpy(at, idx + j, 32);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) at[e] = idx[min(j + e, n - 1)];
    }
    const int first = __builtin_amdgcn_readfirstlane(at[0]);
    const int last = __builtin_amdgcn_readlane(at[7], 63);
    const uint16_t* const src = p.k + ((int64_t)bg * D + d0) * p.S;
    uint16_t* const dst = p.k_out + ((int64_t)bg * D + d0) * p.So + j;
    // rows of whole 16-byte pieces are read at their boundaries
    const int s0 = p.S % 8 == 0 ? first & ~7 : first;
    const int len = last + 1 - s0;
    auto rows_of = [&](auto np) {
      move_rows<decltype(np)::value>(p, src, dst, rows, at, s0, len, j, n, lane, s_win[wave]);
    };
    if (len <= 512) rows_of(std::integral_constant<int, 1>{});
    else if (len <= 1024) rows_of(std::integral_constant<int, 2>{});
    else if (len <= 2048) rows_of(std::integral_constant<int, 4>{});
    else if (len <= kMoveWin) rows_of(std::integral_constant<int, 8>{});
    else move_far(p, src, dst, rows, at, s0, last, j, n, lane, s_win[wave]);
    return;
  }
  x -= p.nk;
  const int j0 = x * p.slots_v, jn = min(p.slots_v, n - j0);
  if (jn <= 0) return;
  if (tid < jn) p.w_out[(int64_t)bg * p.So + j0 + tid] = p.w[(int64_t)bg * p.S + idx[j0 + tid]];
  // eight pieces of a thread at a time, 256 apart
  const int cpr = D / 8, end = jn * cpr;
  const uint16_t* const src = p.v + (int64_t)bg * p.S * D;
  uint16_t* const dst = p.v_out + ((int64_t)bg * p.So + j0) * D;
  for (int e0 = tid; e0 < end; e0 += 8 * 256) {
    int64_t from[8];
    u32x4_t v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int e = min(e0 + 256 * u, end - 1), j = e / cpr;
      from[u] = (int64_t)idx[j0 + j] * D + (e - j * cpr) * 8;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const u32x4_t*>(src + from[u]);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (e0 + 256 * u < end)
        store_stream(reinterpret_cast<u32x4_t*>(dst + (int64_t)(e0 + 256 * u) * 8), v[u]);
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

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
  const int64_t cache = B * G * S * D * 2, added = B * T * G * D * 2;
  const LoomSpan in[] = {{new_k, added}, {new_v, added}, {lens, B * 4}, {counts, B * 4}},
                 out[] = {{k, cache}, {v, cache}, {weights, B * G * S * 4}, {lens_out, B * 4}};
  if (loom_outputs_overlap(in, out))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_append: k, v, weights and lens_out must not overlap the other tensors "
                     "or each other");
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
  // a thread per element up to three tokens (B32 G8 D128, one token: 3.6 us
  // against 4.6 in tiles; two 4.0 and 4.6), tiles above (four 4.8 and 4.6, 16
  // 7.7 and 6.8, 64 16.5 and 8.5)
  if (T < 4) {
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
  const LoomSpan in[] = {{k, kin}, {v, kin}, {weights, B * G * S * 4}, {lens, B * 4}},
                 out[] = {{k_out, kout}, {v_out, kout}, {weights_out, B * G * S_out * 4},
                          {lens_out, B * 4}, {index, B * G * keep * 4}};
  if (loom_outputs_overlap(in, out))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_evict: outputs must not overlap the inputs or each other");
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
  auto select = [&](auto kern) { hipLaunchKernelGGL(kern, sel, selb, 0, st, p); };
  if (S <= 2 * kSel) select(cache_select_kernel<2>);
  else if (S <= 4 * kSel) select(cache_select_kernel<4>);
  else if (S <= 8 * kSel) select(cache_select_kernel<8>);
  else if (S <= 16 * kSel) select(cache_select_kernel<16>);
  else if (S <= 32 * kSel) select(cache_select_kernel<32>);
  else select(cache_select_kernel<0>);
  int rc = loom_check_launch(err, errlen, "cache_evict (select)");
  if (rc) return rc;
  // rows of a K part's wave: as many (two to four) as leave about 4096 waves
  // (B8 G8 S16383: four rows 79.2 us a call, eight 80.3, sixteen 85.8, two 89.3);
  // one or two where the kept slots of a full cache are spread over several windows,
  // which a wave takes one after another (B8 G8 S16383 -> 1024: four rows 99.6, two
  // 66.5; B32 S16384 -> 512: two 54.2, one 42.7)
  p.njk = (int)cdiv64(keep, kMoveJ);
  const bool far = S >= kMoveWin / kMoveJ * keep;
  p.rows_k = (int)std::max<int64_t>(
      far ? 1 : 2, std::min<int64_t>(far ? 2 : 4, B * G * p.njk * D / 4096));
  p.nk = (int)(p.njk * cdiv64(D, 4 * p.rows_k));
  // slots of a V part: eight 16-byte pieces a thread, fewer for about 1024 parts
  p.slots_v = (int)std::max<int64_t>(
      8, std::min({(int64_t)256, 16384 / D, cdiv64(B * G * keep, 1024)}));
  const dim3 grid((unsigned)(p.nk + cdiv64(keep, p.slots_v)), (unsigned)(B * G));
  hipLaunchKernelGGL(cache_move_kernel, grid, dim3(256), 0, st, p);
  return loom_check_launch(err, errlen, "cache_evict (move)");
}

}  // extern "C"
