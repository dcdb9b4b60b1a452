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
//
// gfx950 mapping.  A prompt reads 2 (H D + D + E) and writes 2 H E bytes a token and KV
// head for 4 H D E operations: bound by HBM where the states stay on the chip, as they do
// here, in the accumulators of the waves that walk a head's chunks (linear_chunk_kernel).
// Where heads are fewer than CUs the tokens are cut into segments: a first launch leaves
// the segments' states, from k and v alone, a second one walks every segment
// from the sum of those before it.  One token is a stream of the states, read and written
// once (linear_step_kernel).
#include "common.h"

#include <cmath>
#include <type_traits>

namespace {

constexpr int kC = 32;            // tokens of a chunk
constexpr int kIT = kC / 16;      // tiles of queries

struct LinearParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const float* g;        // log decays
  const float* state;
  const int* counts;
  uint16_t* out;
  float* state_out;
  float* ws;             // [B G H, nseg, D, E]: the initial states and those of segments
  int B, G, H, D, E, T;
  int nsl;               // slices of E
  int nseg;              // segments of a prompt
  int cps;               // chunks of a segment
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
// a s + x: an infinite s stays what it is (its product with lo would be NaN, or the other
// infinity); one more instruction, which a step's stream of states hides
LOOM_DEV float decayed_plus(float s, const Decay& a, float x) {
  const float f = __builtin_amdgcn_fmed3f(s, -__FLT_MAX__, __FLT_MAX__);
  return __builtin_fmaf(s, a.hi, __builtin_fmaf(f, a.lo, x));
}

// A row's 16-byte chunks are XORed with this, so that both the 16 rows of a direct read
// of q or k (one chunk each) and the 8 consecutive rows of a pass of v's transposed reads
// (a pair of chunks each) lie on distinct banks: rows of 128 bytes and of multiples of 256.
// k's transposed reads take four chunks of a row, two of which share banks (40 to 47% of
// the kernel's LDS cycles): reads without these conflicts took 32 more vector instructions
// a chunk, and longer (32768 tokens 395 us against 375 in the version they were tried in).
template <int N>
LOOM_DEV int row_swz(int row) {
  return (N >= 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3)) ^ ((row >> 3) & 1);
}

// 2^k, |k| < 127
LOOM_DEV float pow2i(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }
// A power of two that brings the largest finite magnitude of a wave's values to 2^13:
// f16 operands beyond 65504, or below 2^-14 throughout, would lose what fp32 holds.
// m: this lane's largest magnitude.
LOOM_DEV float f16_scale(float m) {
  m = wave_max(m);
  const int e = max(-60, (int)(__float_as_uint(m) >> 23) - 127);
  return pow2i(13 - e);
}
// the largest magnitude, NaN if one is NaN
LOOM_DEV float largest(float x, float y, float z) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(fabsf(y), fabsf(z)), x);
}
// What keeps a NaN once one of eight 16-bit numbers was infinite or NaN (bf16: or beyond
// 2^121), two numbers at a time.  Infinite and NaN bf16 bits are NaN as f16.
template <bool F16>
LOOM_DEV f16x2_t odd16(f16x2_t odd, const u32x4_t& x) {
  // (by value: a cast of an element of the vector itself reads the first one)
  auto half2 = [](uint32_t w) { return __builtin_bit_cast(f16x2_t, w); };
  if constexpr (F16) {
    const f16x2_t zero = f16x2_t{0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) odd = __builtin_elementwise_fma(half2(x[i]), zero, odd);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i += 2)
      odd = __builtin_elementwise_maximum(__builtin_elementwise_maximum(odd, half2(x[i])),
                                          half2(x[i + 1]));
  }
  return odd;
}
// ones in the halves of w that are neither infinite nor NaN (an exponent of all ones carries
// into the sign's place)
template <bool F16>
LOOM_DEV uint32_t finite16(uint32_t w) {
  const uint32_t inf = F16 ? 0x7c007c00u : 0x7f807f80u, one = F16 ? 0x04000400u : 0x00800080u;
  return ~(((((w & inf) + one) & 0x80008000u) >> 15) * 0xffffu);
}
LOOM_DEV float finite_abs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }

// The same address in every lane, stated to the compiler
LOOM_DEV const char* uniform(const char* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const char*>(
      ((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32) |
      (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v));
}

// Chunked form.  A workgroup of W waves walks the chunks of 32 tokens of one (b, g, h)
// and 16 W columns of E in order, each wave holding the state's D x 16 columns in the
// accumulators of its MFMAs, fp32.  For a chunk of tokens 0 .. C-1 and the state S before
// it:
//   P_ij = scale a^(i-j) q_i.k_j (j <= i),
//   out_i = sum_j P_ij v_j + scale a^(i+1) S^T q_i,
//   S' = a^C S + sum_j k_j (a^(C-1-j) v_j)^T.
// The MFMAs compute transposed tiles, S^T[e, d] . Q^T[d, i] and V^T[e, j] . P^T[j, i], so
// that a wave's state feeds the first product from its own accumulators: the state's row
// tiles are taken so that lane group g holds d = 32 t + 8 g + 0..7 in a pair of them, the
// 16 bytes of q that it reads.  P^T is built from the accumulators of K Q^T, one chunk
// ahead, by four waves (in f16 two), and shared through LDS: one barrier to a chunk.
// Rounding: S and P to 16 bits as operands, each once; a^(C-1-j) v_j as a sum of three
// bf16 or two f16 numbers, so that the state keeps fp32's accuracy (f16: to 2^-36 of k
// where v is below 2^-14).  f16 operands are scaled by powers of two where they leave its
// range.
// What bounds it: a chunk of 128 x 128 takes a CU 1.4 us by itself (24 + 8 products of 16
// cycles and 200 other vector instructions to each of 8 waves), its 32 KB 1.6 us at the
// rate of a large copy.  B8 G32 of 1024 to 4096 tokens 195 to 206 us (738 MB, 3.7 TB/s: the
// longest prompt's 128 chunks in a row, while the CUs of shorter ones idle), B1 G32 of
// 32768 370 to 395 us (1.08 GB, and k, v once more in the first launch, 0.47 GB); key dims
// of 256: B4 G32 256 x 256 T2048 189 us, in f16 274.  Measured while
// it was built, at B8 G32: chunks of 64 tokens by four waves 366 us, by eight 249 (the 64 x
// 64 scores cost more than they save); of 32 by four waves of 32 columns 251 to 257, by
// eight of 16 216; then direct reads of 16 bytes (not two of 8, which the compiler joined
// and took apart again by moves) and one branch to a chunk's copies 201, and k's transposed
// reads without their bank conflicts 206.  A fourth stage: no change.
// Infinities and NaN: every chunk is looked over while the one before it is worked on; one
// that holds any, other than for states lost to NaN already, is taken token by token
// (by_token), by the recurrence itself, for about 14 us.
// ONLY_STATE: a segment's own state from zero (the first's from the initial state), which
// later segments start from.
template <int DK, int W, bool F16, bool ONLY_STATE>
__global__ void __launch_bounds__(64 * W, (ONLY_STATE ? DK < 256 : DK == 64 && !F16) ? 4 : 2)
    linear_chunk_kernel(LinearParams p) {
  constexpr int SL = 16 * W;                    // columns of a workgroup
  constexpr int KROW = DK * 2, VROW = SL * 2;
  constexpr int Q_BYTES = ONLY_STATE ? 0 : kC * KROW, K_BYTES = kC * KROW, V_BYTES = kC * VROW;
  constexpr int STAGE = Q_BYTES + K_BYTES + V_BYTES;
  // stages: this chunk, the next (whose P^T is built) and the one on its way (a fourth
  // took as long)
  constexpr int NS = 3;
  constexpr int KS = DK / 32, DT = DK / 16;
  constexpr int TERMS = F16 ? 2 : 3;            // 16-bit numbers that hold a^(C-1-j) v_j
  static_assert(kC == 32, "one step of the MFMA over a chunk's tokens");
  static_assert(V_BYTES / W == 1024, "a copy of v to each wave");
  __shared__ __attribute__((aligned(1024))) char smem[NS * STAGE];
  __shared__ __attribute__((aligned(16))) u32x4_t s_p[ONLY_STATE ? 1 : 2 * kIT * 64];
  __shared__ float s_pow[kC + 1];
  __shared__ float s_ps[2][kIT];                // f16: what a tile of P was scaled by
  // the last chunks found to hold infinities or NaN, and to hold them in q or k
  __shared__ int s_odd[2], s_keys[2];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g4 = lane >> 4;
  const int a4 = r >> 2, c4 = r & 3;
  // (b, g) outermost, then segments, heads, slices: those that share k and v side by side
  const int nsl = p.nsl, H = p.H, D = p.D, E = p.E, GH = p.G * H;
  const int nseg = ONLY_STATE ? p.nseg - 1 : p.nseg;
  int id = xcd_remap(blockIdx.x, gridDim.x);
  const int sl = id % nsl;
  id /= nsl;
  const int h = id % H;
  id /= H;
  const int seg = id % nseg, bg = id / nseg;
  const int b = bg / p.G, g = bg - b * p.G, gh = g * H + h;
  const int c =
      __builtin_amdgcn_readfirstlane(p.counts ? min(max(p.counts[b], 0), p.T) : p.T);
  const int64_t seglen = (int64_t)p.cps * kC;
  const int t0 = (int)(seg * seglen);           // (T < 2^29 and a segment within T)
  // a segment's state is asked for by those behind it only
  const bool wanted = !ONLY_STATE || (seg + 1) * seglen < c;
  if (seg > 0 && (!wanted || t0 >= c)) return;
  const int tokens = wanted ? (int)min((int64_t)(c - t0), seglen) : 0;
  const int nch = (tokens + kC - 1) / kC;

  // ---- copies of chunk ci into a stage: rows past the sequence and chunks past D or E
  // from zeros.  A whole chunk of whole rows takes each copy as the chunk's scalar base
  // plus this lane's offset, computed once (fast: all offsets fit 32 bits).
  const int64_t tok0 = (int64_t)b * p.T + t0;
  const uint16_t* const qb = p.q + (tok0 * GH + gh) * D;
  const uint16_t* const kb = p.k + (tok0 * p.G + g) * D;
  const uint16_t* const vb = p.v + (tok0 * p.G + g) * E + sl * SL;
  // token strides in bytes (at most 2^29)
  const uint32_t qs = (uint32_t)(GH * D * 2), ks_ = (uint32_t)(p.G * D * 2),
                 vs = (uint32_t)(p.G * E * 2);
  const bool fast = D == DK && sl * SL + SL <= E && qs < (1u << 26) && vs < (1u << 26);
  // copies of a row of N elements times 32 tokens, 1 KB each, which the waves share (the
  // last ones of fewer than W go to some of them)
  constexpr int QK_ALL = K_BYTES / 1024, QK_INSTR = (QK_ALL + W - 1) / W;
  uint32_t qoff[QK_INSTR], koff[QK_INSTR], voff[1];
  auto offsets = [&](auto& off, uint32_t stride, auto n) {
    constexpr int N = decltype(n)::value, ALL = kC * N * 2 / 1024, INSTR = (ALL + W - 1) / W;
#pragma unroll
    for (int i = 0; i < INSTR; ++i) {
      const int e = (wave + W * i) * 64 + lane, row = e / (N / 8);
      off[i] = row * stride + ((e % (N / 8)) ^ row_swz<N>(row)) * 16;
    }
  };
  using QK = std::integral_constant<int, DK>;
  using VC = std::integral_constant<int, SL>;
  offsets(qoff, qs, QK{});
  offsets(koff, ks_, QK{});
  offsets(voff, vs, VC{});
  // where the next chunk to be copied begins, and how many tokens are left there
  const char *qat = reinterpret_cast<const char*>(qb), *kat = reinterpret_cast<const char*>(kb),
             *vat = reinterpret_cast<const char*>(vb);
  int ahead = tokens;
  const uint32_t lds0 = lds_addr((lds_char_t*)smem) + wave * 1024;
  auto issue = [&](int s) {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + s * STAGE);
    if (fast && ahead >= kC) {                  // wave-uniform
      auto rows = [&](const char* at, auto& off, auto n, uint32_t lds) {
        constexpr int N = decltype(n)::value, ALL = kC * N * 2 / 1024, INSTR = (ALL + W - 1) / W;
        at = uniform(at);
#pragma unroll
        for (int i = 0; i < INSTR; ++i) {
          if (ALL % W && wave + W * i >= ALL) break;
          dma_load16_s(off[i], at, lds + W * i * 1024);
        }
      };
      if constexpr (!ONLY_STATE) rows(qat, qoff, QK{}, to);
      rows(kat, koff, QK{}, to + Q_BYTES);
      rows(vat, voff, VC{}, to + Q_BYTES + K_BYTES);
    } else {
      auto rows = [&](const char* at, uint32_t stride, int valid, auto n, uint32_t lds) {
        constexpr int N = decltype(n)::value, ALL = kC * N * 2 / 1024, INSTR = (ALL + W - 1) / W;
        const int ln = fresh(lane);
#pragma unroll
        for (int i = 0; i < INSTR; ++i) {
          const int j = wave + W * i;
          if (ALL % W && j >= ALL) break;
          const int e = j * 64 + ln, row = e / (N / 8), ch = (e % (N / 8)) ^ row_swz<N>(row);
          const void* src = row < ahead && ch < valid
                                ? (const void*)(at + (int64_t)row * stride + ch * 16)
                                : (const void*)(loom_zero_kb + lane * 4);
          dma_load16(src, __builtin_amdgcn_readfirstlane(lds + W * i * 1024));
        }
      };
      if constexpr (!ONLY_STATE) rows(qat, qs, D / 8, QK{}, to);
      rows(kat, ks_, D / 8, QK{}, to + Q_BYTES);
      rows(vat, vs, (E - sl * SL) / 8, VC{}, to + Q_BYTES + K_BYTES);
    }
    qat += (int64_t)kC * qs;
    kat += (int64_t)kC * ks_;
    vat += (int64_t)kC * vs;
    ahead -= kC;
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (i < nch) issue(i);

  const float lg = p.g[gh];
  if (tid <= kC) s_pow[tid] = (float)decay_pow(lg, tid);
  if (tid < 2) s_odd[tid] = s_keys[tid] = -1;
  Decay one = split_decay(decay_pow(lg, 1));
  one.hi = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(one.hi)));
  one.lo = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(one.lo)));
  // Powers that fp32 holds as zero are its smallest number where the decay is not zero, so
  // that an infinite state stays infinite; a finite one is then 2^-149 of itself, not zero.
  const float least = __uint_as_float(one.hi > 0.f ? 1u : 0u);
  // over a whole chunk, and over the last one.  A rounded factor near 1, applied over and
  // over, would be off by its rounding times the chunks that a head remembers: what the
  // factors so far are off by (relatively) is kept, and each makes up for it.
  Decay full = split_decay(decay_pow(lg, kC));
  Decay last = split_decay(decay_pow(lg, tokens - (nch - 1) * kC));
  full.hi = fmaxf(full.hi, least);
  last.hi = fmaxf(last.hi, least);
  const float inv_full = full.hi > 1e-30f ? 1.f / full.hi : 0.f;
  float owed = 0.f;

  // ---- the state: s[dt][i] is row d = 32 (dt / 2) + 8 g4 + 4 (dt % 2) + i, column ec.  By
  // buffer accesses, which the hardware checks against the state's end: rows past D and
  // columns past E read as zeros and are not written.
  const int col0 = sl * SL + wave * 16, ec = col0 + r;
  f32x4_t s[DT];
  const int64_t bgh = (int64_t)b * GH + gh, sz = (int64_t)D * E;
  const uint32_t sbytes = (uint32_t)(D * E * 4);
  const uint32_t sbase = ec < E ? (uint32_t)(8 * g4 * E + ec) * 4 : 1u << 30;
  auto at_state = [&](int dt, int i) {
    return sbase + (uint32_t)((32 * (dt >> 1) + 4 * (dt & 1) + i) * E) * 4;
  };
  auto read_state = [&](const float* from, f32x4_t (&x)[DT]) {
    const rsrc_t rs = make_rsrc(from, sbytes);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[dt][i] = __uint_as_float(buf_load4(rs, at_state(dt, i)));
  };
  auto write_state = [&](float* to) {
    const rsrc_t rs = make_rsrc(to, sbytes);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s[dt][i]), rs, at_state(dt, i), 0, 0);
  };
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) s[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // the first launch's states: slot 0 the initial one (state_out may be state: the first
  // segment reads this copy), slot u + 1 that of segment u
  const int64_t slots = p.nseg;
  if (p.nseg == 1 || (ONLY_STATE && seg == 0)) {
    if (p.state) read_state(p.state + bgh * sz, s);
    if constexpr (ONLY_STATE) write_state(p.ws + bgh * slots * sz);
  } else if constexpr (!ONLY_STATE) {
#pragma unroll 1
    for (int u = seg == 0 ? 0 : 1; u <= seg; ++u) {
      const float w = fmaxf((float)exp((double)(seg - u) * (double)seglen *
                                       (double)(lg < -1e30f ? -1e30f : lg)),
                            least);
      f32x4_t x[DT];
      read_state(p.ws + (bgh * slots + u) * sz, x);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) s[dt] += x[dt] * w;
    }
  }

  // ---- factors, the same for every whole chunk.  An operand's eight tokens of lane group
  // g4: 4 g4 + 0..3 and 16 + 4 g4 + 0..3
  __syncthreads();          // (s_pow)
  auto token = [&](int x) { return 16 * (x >> 2) + 4 * g4 + (x & 3); };
  float w[8], rise[kIT];
#pragma unroll
  for (int x = 0; x < 8; ++x) w[x] = s_pow[kC - 1 - token(x)];
#pragma unroll
  for (int it = 0; it < kIT; ++it) rise[it] = fmaxf(p.scale * s_pow[16 * it + r + 1], least);
  // A wave's part of P^T: of a tile of queries, the half of 16 tokens, in f16 both (which
  // share what they are scaled by).  Of 8 waves (in f16 4) they take turns.
  const int pit = F16 ? wave & 1 : (wave >> 1) & 1, pt = F16 ? 0 : wave & 1;
  constexpr int PT = F16 ? 2 : 1, TURNS = W * PT / 4;
  const int turn = wave / (W / TURNS);
  float pf_fac[4 * PT];
  bool seen[4 * PT];
#pragma unroll
  for (int x = 0; x < 4 * PT; ++x) {
    const int lag = 16 * (pit - pt) + r - token(x);
    seen[x] = lag >= 0;
    pf_fac[x] = p.scale * s_pow[max(lag, 0)];
  }
  const char* ob = reinterpret_cast<const char*>(p.out + (tok0 * GH + gh) * E + col0);
  const int64_t ostep = (int64_t)16 * GH * E * 2;
  const int64_t ooff = (int64_t)r * GH * E * 2 + 8 * g4;
  const bool stores = !ONLY_STATE && col0 < E;
  // stores of a chunk's rows, all of which a whole chunk issues
  constexpr int STORES = kIT;

  // rows 16 t + r of q or k, elements d = 32 ks + 8 g4 .. + 7
  auto row_op = [&](const lds_char_t* base, int t, int ks) {
    const int row = 16 * t + r;
    return *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(
        base + row * KROW + ((4 * ks + g4) ^ row_swz<DK>(row)) * 16);
  };
  // sixteen columns of K or V, transposed; chunk and half: where this lane's four of them
  // lie in a row
  auto col_op = [&](const lds_char_t* base, auto n, int chunk, int half) {
    constexpr int N = decltype(n)::value;
    const int row = 4 * g4 + a4;
    const lds_char_t* at = base + row * (N * 2) + (chunk ^ row_swz<N>(row)) * 16 + half * 8;
    const u32x2_t lo = lds_read_tr16(at);
    const u32x2_t hi = lds_read_tr16(at + 16 * (N * 2));    // (the same swizzle)
    return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
  };
  // P^T of chunk ci in a stage, as the operands that every wave reads, into s_p[ci & 1]
  auto build_p = [&](const lds_char_t* st, int ci) {
    const int to = ci & 1;
    f32x4_t x[PT] = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const u32x4_t q = row_op(st, pit, ks);
#pragma unroll
      for (int t = 0; t < PT; ++t) x[t] = mfma16t<F16>(row_op(st + Q_BYTES, pt + t, ks), q, x[t]);
    }
    // an infinity or NaN of q or k makes all its scores so, those of tokens not seen too
    float big = 0.f;
#pragma unroll
    for (int t = 0; t < PT; ++t) big = largest(largest(big, x[t][0], x[t][1]), x[t][2], x[t][3]);
    if (__builtin_amdgcn_ballot_w64(!(big < INFINITY)) != 0 && lane == 0)
      s_odd[to] = s_keys[to] = ci;
#pragma unroll
    for (int t = 0; t < PT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = x[t][e] * pf_fac[4 * t + e];
        x[t][e] = seen[4 * t + e] ? y : 0.f;
      }
    if constexpr (F16) {
      float mx = 0.f;
#pragma unroll
      for (int t = 0; t < PT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, finite_abs(x[t][e]));
      const float sc = f16_scale(mx);
#pragma unroll
      for (int t = 0; t < PT; ++t) x[t] *= sc;
      if (lane == 0) s_ps[to][pit] = sc;
    }
#pragma unroll
    for (int t = 0; t < PT; ++t)
      reinterpret_cast<u32x2_t*>(&s_p[(to * kIT + pit) * 64 + lane])[pt + t] =
          u32x2_t{pack2<F16>(x[t][0], x[t][1]), pack2<F16>(x[t][2], x[t][3])};
  };
  // Whether chunk ci in a stage holds infinities or NaN: of k and v (without scores; a piece
  // of each to a wave), or of v, by the waves whose turn at P^T comes next.  A chunk ahead,
  // so that its work has no branch in its midst, which took 8% (the checks take 1 to 2).
  constexpr int PIECES = ONLY_STATE ? QK_INSTR + 1 : TURNS;
  u32x4_t held[PIECES];
  auto peek = [&](const lds_char_t* st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      int at = QK_ALL + (ONLY_STATE ? wave : (wave - turn * (W / TURNS)) * TURNS + i);
      if (ONLY_STATE && i < QK_INSTR) at = min(wave + W * i, QK_ALL - 1);
      held[i] = *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(
          st + Q_BYTES + at * 1024 + lane * 16);
    }
  };
  auto judge = [&](int ci) __attribute__((always_inline)) {
    auto any = [&](int from, int to) {
      f16x2_t odd = f16x2_t{0, 0};
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        if (i >= from && i < to) odd = odd16<F16>(odd, held[i]);
      return __builtin_amdgcn_ballot_w64(odd[0] != odd[0] || odd[1] != odd[1]) != 0;
    };
    if (any(0, PIECES)) {
      const bool keys = ONLY_STATE && any(0, PIECES - 1);
      if (lane == 0) {
        s_odd[ci & 1] = ci;
        if (keys) s_keys[ci & 1] = ci;
      }
    }
  };
  if (nch > 0) {
    LOOM_WAIT_VMCNT(0);
    barrier_nofence();
    const lds_char_t* const st = (lds_char_t*)smem;
    if constexpr (!ONLY_STATE)
      if (turn == 0) build_p(st, 0);
    if (ONLY_STATE || turn == TURNS - 1) {
      peek(st);
      judge(0);
    }
  }
  // A chunk that holds an infinity or NaN, token by token as the recurrence has it, in
  // fp32: products with zeros and with the numbers that v is split into would make NaN of
  // infinities, and reach rows ahead of theirs.  Returns which of this lane's outputs are
  // infinite or NaN: a bit each, 8 for inf, 8 for -inf, 8 for NaN.
  auto by_token = [&](const lds_char_t* st, int n) __attribute__((always_inline)) {
    uint32_t bad = 0;
    const int ln = fresh(lane), r = ln & 15, g4 = ln >> 4;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const lds_char_t* const kr = st + Q_BYTES + j * KROW;
      const lds_char_t* const vr = st + Q_BYTES + K_BYTES + j * VROW;
      typedef const __attribute__((address_space(3))) uint16_t* at16_t;
      typedef const __attribute__((address_space(3))) u32x2_t* at64_t;
      const float v = lo16<F16>(*reinterpret_cast<at16_t>(
          vr + ((wave * 2 + (r >> 3)) ^ row_swz<SL>(j)) * 16 + (r & 7) * 2));
      float o = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int at = ((4 * (dt >> 1) + g4) ^ row_swz<DK>(j)) * 16 + 8 * (dt & 1);
        const u32x2_t k = *reinterpret_cast<at64_t>(kr + at);
        u32x2_t q = u32x2_t{0u, 0u};
        if constexpr (!ONLY_STATE)
          q = *reinterpret_cast<at64_t>(st + j * KROW + at);
        lds_order();      // (one tile's reads at a time: registers)
        if (32 * (dt >> 1) + 8 * g4 >= D) continue;     // (rows past D stay zeros)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float ki = i & 1 ? hi16<F16>(k[i >> 1]) : lo16<F16>(k[i >> 1]);
          s[dt][i] = decayed_plus(s[dt][i], one, ki * v);
          if constexpr (!ONLY_STATE)
            o = __builtin_fmaf(s[dt][i], i & 1 ? hi16<F16>(q[i >> 1]) : lo16<F16>(q[i >> 1]), o);
        }
      }
      if constexpr (!ONLY_STATE) {
        // (which part of a sum over d was infinite or NaN tells what it is)
        auto columns = [](bool is) {
          const uint64_t m = __builtin_amdgcn_ballot_w64(is), x = m | m >> 32;
          return (uint32_t)(x | x >> 16) & 0xffffu;
        };
        const uint32_t pos = columns(o == INFINITY), neg = columns(o == -INFINITY);
        const uint32_t nan = columns(o != o) | (pos & neg);
        if (r == (j & 15))                              // columns 4 g4 .. + 3 of token j
          bad |= ((pos >> 4 * g4 & 15u) | (neg >> 4 * g4 & 15u) << 8 | (nan >> 4 * g4 & 15u) << 16)
                 << 4 * (j >> 4);
      }
    }
    return bad;
  };
  int stage = 0;
  // (one of each for both kinds of chunks: as their own, the kernels of D 256 spill)
  f32x4_t o[kIT];
  u32x4_t vf;               // v as an operand
  // ---- S^T Q^T of the state before a chunk, times scale a^(i+1), into o.  Products that
  // wait for each other are kept apart; between: what is worked out among them, in fours
  auto ahead_of = [&](const lds_char_t* lq, auto between) __attribute__((always_inline)) {
    float sc = 1.f;
    if constexpr (F16) {
      float mx = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, finite_abs(s[dt][i]));
      sc = f16_scale(mx);
    }
    const float back = F16 ? 1.f / sc : 1.f;
#pragma unroll
    for (int it = 0; it < kIT; ++it) o[it] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      f32x4_t x = s[2 * ks], y = s[2 * ks + 1];
      if constexpr (F16) {
        x *= sc;
        y *= sc;
      }
      const u32x4_t sp = u32x4_t{pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]),
                                 pack2<F16>(y[0], y[1]), pack2<F16>(y[2], y[3])};
#pragma unroll
      for (int it = 0; it < kIT; ++it) o[it] = mfma16t<F16>(sp, row_op(lq, it, ks), o[it]);
#pragma unroll
      for (int y4 = 4 * ks / KS; y4 < 4 * (ks + 1) / KS; ++y4) between(y4);
    }
#pragma unroll
    for (int it = 0; it < kIT; ++it)
      o[it] *= F16 ? fmaxf(rise[it] * back, least) : rise[it];
  };
  // ---- V^T P^T of the chunk's own tokens, and its outputs
  auto finish = [&](int ci, auto is_odd, uint32_t bad) __attribute__((always_inline)) {
    const int left = tokens - ci * kC;
#pragma unroll
    for (int it = 0; it < kIT; ++it) {
      const u32x4_t pf = s_p[((ci & 1) * kIT + it) * 64 + lane];
      const float ps = F16 ? s_ps[ci & 1][it] : 1.f;
      if constexpr (F16) o[it] *= ps;
      o[it] = mfma16t<F16>(vf, pf, o[it]);
      if constexpr (F16) o[it] *= 1.f / ps;
      if constexpr (decltype(is_odd)::value) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t is = bad >> (4 * it + e);
          o[it][e] = is & 0x10000u ? NAN : is & 1u ? INFINITY : is & 0x100u ? -INFINITY : o[it][e];
        }
      }
      // ---- o[it][e] is token 16 it + r, column col0 + 4 g4 + e
      char* to = const_cast<char*>(uniform(ob)) + ooff;
      ob += ostep;
      if (16 * it + r < left && col0 + 4 * g4 < E)
        *(__attribute__((address_space(1))) u32x2_t*)to =
            u32x2_t{pack2<F16>(o[it][0], o[it][1]), pack2<F16>(o[it][2], o[it][3])};
    }
  };
  // Whether by_token has to take the chunk, which holds infinities or NaN of q or k (keys)
  // or of v: not where these only meet columns whose states are all NaN already, and stay so
  // (else whatever follows a NaN would take as long).
  auto matters = [&](const lds_char_t* lv, bool keys) __attribute__((always_inline)) {
    const int g4 = fresh(lane) >> 4;
    bool lost = true;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) lost &= s[dt][i] != s[dt][i] || 32 * (dt >> 1) + 8 * g4 >= D;
    const f16x2_t x =
        odd16<F16>(f16x2_t{0, 0}, col_op(lv, VC{}, wave * 2 + (c4 >> 1), c4 & 1));
    // a bit to each of the wave's columns, all of whose four lanes, or one of them
    auto fold = [](uint64_t m) {
      m |= m >> 32;
      return (uint32_t)(m | m >> 16) & 0xffffu;
    };
    const uint32_t live = fold(__builtin_amdgcn_ballot_w64(!lost && ec < E)),
                   odd = fold(__builtin_amdgcn_ballot_w64(x[0] != x[0] || x[1] != x[1]));
    return (live & (keys ? 0xffffu : odd)) != 0;
  };
  // The start of chunk ci: its copies have landed, those of chunk ci + 2 set out, and chunk
  // ci + 1's scores are built.  Returns whether by_token has to take it.
  lds_char_t* lq = nullptr;         // where the chunk lies
  float a = 0.f;                    // its decay
  auto begin = [&](int ci) __attribute__((always_inline)) {
    const int left = tokens - ci * kC;
    lq = (lds_char_t*)(smem + stage * STAGE);
    lds_order();
    // the copies of the next chunk; the stores of the one before are younger
    if (stores && ci > 0) LOOM_WAIT_VMCNT(STORES);
    else LOOM_WAIT_VMCNT(0);
    LOOM_WAIT_LGKM0();
    barrier_nofence();
    const int flag = s_odd[ci & 1];
    const lds_char_t* const next = (lds_char_t*)(smem + (stage == NS - 1 ? 0 : stage + 1) * STAGE);
    if constexpr (ONLY_STATE) peek(next);         // (judged below: behind the copies' start)
    if (ci + NS - 1 < nch) issue(stage == 0 ? NS - 1 : stage - 1);
    stage = stage == NS - 1 ? 0 : stage + 1;
    a = __builtin_fmaf(full.hi, owed, full.hi);
    owed = __builtin_fmaf((full.hi - a) + full.lo, inv_full, owed);
    if (left < kC) {          // the last, partial chunk
      a = __builtin_fmaf(last.hi, owed, last.hi);
      const int j0 = fresh(4 * g4);
#pragma unroll
      for (int x = 0; x < 8; ++x) w[x] = s_pow[max(0, left - 1 - (16 * (x >> 2) + j0 + (x & 3)))];
    }
    if (ci + 1 < nch) {
      if constexpr (!ONLY_STATE) {
        if (turn == (ci + 1) % TURNS) build_p(next, ci + 1);
        if (turn == (ci + 2) % TURNS) {
          peek(next);
          judge(ci + 1);
        }
      } else {
        judge(ci + 1);
      }
    }
    if (__builtin_amdgcn_readfirstlane(flag) != ci) return false;
    return matters(lq + Q_BYTES + K_BYTES,
                   __builtin_amdgcn_readfirstlane(s_keys[ci & 1]) == ci);
  };
  // A chunk without infinities or NaN that matter
  auto usual = [&](int ci) __attribute__((always_inline)) {
    const lds_char_t *const lk = lq + Q_BYTES, *const lv = lk + K_BYTES;

    // ---- v as an operand, and a^(C-1-j) v as a sum of 16-bit numbers
    vf = col_op(lv, VC{}, wave * 2 + (c4 >> 1), c4 & 1);
    u32x4_t vt[TERMS];
    // f16: the second number 2^11 times larger, in sums of its own, so that it keeps
    // its bits
    constexpr float kLow = F16 ? 2048.f : 1.f;
    auto weigh = [&](int x) {
      float y0 = lo16<F16>(vf[x]) * w[2 * x], y1 = hi16<F16>(vf[x]) * w[2 * x + 1];
#pragma unroll
      for (int z = 0; z < TERMS; ++z) {
        const uint32_t y = pack2<F16>(y0, y1);
        vt[z][x] = y;
        if (z + 1 < TERMS) {
          y0 = (y0 - lo16<F16>(y)) * kLow;
          y1 = (y1 - hi16<F16>(y)) * kLow;
        }
      }
    };

    if constexpr (!ONLY_STATE) {
      ahead_of(lq, weigh);
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) weigh(x);
    }

    // ---- the state behind the chunk, row tiles in fours
#pragma unroll
    for (int d4 = 0; d4 < DT; d4 += 4) {
      u32x4_t kt[4];
      f32x4_t x[4], y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        kt[u] = col_op(lk, QK{}, 2 * (d4 + u - (u & 1)) + c4, u & 1);
        x[u] = y[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int z = TERMS - 1; z >= 0; --z)      // the small ones first
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          f32x4_t& t = F16 && z == 1 ? y[u] : x[u];
          t = mfma16t<F16>(kt[u], vt[z], t);
        }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float z = F16 ? __builtin_fmaf(y[u][i], 1.f / kLow, x[u][i]) : x[u][i];
          s[d4 + u][i] = __builtin_fmaf(s[d4 + u][i], a, z);
        }
      // (stated where the compiler would otherwise put these sums off to the next chunk, and
      // keep their operands in registers that it does not have: D 256 spilled, and took
      // 297 us where it takes 196 at B4 G32 T2048)
      if constexpr (DK == 256 && !ONLY_STATE)
#pragma unroll
        for (int u = 0; u < 4; ++u) asm volatile("" : "+v"(s[d4 + u]));
    }
    if constexpr (ONLY_STATE)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) asm volatile("" : "+v"(s[dt]));
    if constexpr (!ONLY_STATE) finish(ci, std::false_type{}, 0);
  };
  // One with some
  auto spoiled = [&](int ci) __attribute__((always_inline)) {
    if constexpr (!ONLY_STATE) ahead_of(lq, [](int) {});
    const uint32_t bad = by_token(lq, min(tokens - ci * kC, kC));
    if constexpr (!ONLY_STATE) {
      vf = col_op(lq + Q_BYTES + K_BYTES, VC{}, wave * 2 + (c4 >> 1), c4 & 1);
#pragma unroll
      for (int x = 0; x < 4; ++x) vf[x] &= finite16<F16>(vf[x]);
      finish(ci, std::true_type{}, bad);
    }
  };
  // The latter in a loop around the others.  (Beside them in one, or with another way out
  // of theirs than at its end, the state would be copied in it.)
  int ci = 0;
  bool go = nch > 0 && !begin(0);
#pragma unroll 1
  while (ci < nch) {
#pragma unroll 1
    while (go) {
      usual(ci);
      go = ++ci < nch;
      if (go) go = !begin(ci);
    }
    if (ci >= nch) break;
    spoiled(ci);
    go = ++ci < nch;
    if (go) go = !begin(ci);
  }
  if constexpr (ONLY_STATE) {
    if (!wanted) return;
    write_state(p.ws + (bgh * slots + seg + 1) * sz);
  } else if (t0 + tokens == c) {      // the segment that the sequence ends in
    write_state(p.state_out + bgh * sz);
  }
}

// One token.  L lanes of four columns to a row of the state, 256 / L rows at once, 16 of
// them in flight to a thread.  The state is stored past the caches: a program's layers
// have more of it than these hold, so it comes from memory the next time (B64 G32 128 x 128,
// three states in turn: 268 MB in 44.9 us, 6.0 TB/s, against 59.4 with ordinary stores; one
// state over and over 44.7 against 40.5).
template <bool F16>
__global__ void __launch_bounds__(256) linear_step_kernel(LinearParams p, int L) {
  __shared__ float s_q[256], s_k[256];
  __shared__ f32x4_t s_o[256];
  const int GH = p.G * p.H, D = p.D, E = p.E;
  const int tid = threadIdx.x, l = tid & (L - 1), grp = tid / L, NG = 256 / L;
  const int sl = blockIdx.x % p.nsl;
  const int64_t bgh = blockIdx.x / p.nsl;
  const int b = (int)(bgh / GH), gh = (int)(bgh - (int64_t)b * GH), g = gh / p.H;
  if (p.counts && p.counts[b] <= 0) return;
  const int e = (sl * L + l) * 4;
  const bool in = e < E;
  float* const at = p.state_out + bgh * D * E + e;
  constexpr int N = 16;       // rows of a thread in flight
  f32x4_t x[N];
  auto load = [&](int d0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = d0 + grp + NG * i;
      if (in && d < D) x[i] = *reinterpret_cast<const f32x4_t*>(at + (int64_t)d * E);
    }
  };
  const int64_t bg = (int64_t)b * p.G + g;
  const uint16_t qd = p.q[bgh * D + min(tid, D - 1)], kd = p.k[bg * D + min(tid, D - 1)];
  const u32x2_t vd = *reinterpret_cast<const u32x2_t*>(p.v + bg * E + min(e, E - 4));
  const float lg = p.g[gh];
  load(0);                    // (behind the small loads, which are waited for alone)
  if (tid < D) {
    s_q[tid] = lo16<F16>(qd) * p.scale;
    s_k[tid] = lo16<F16>(kd);
  }
  const f32x4_t v = f32x4_t{lo16<F16>(vd[0]), hi16<F16>(vd[0]), lo16<F16>(vd[1]), hi16<F16>(vd[1])};
  f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const Decay a = split_decay(decay_pow(lg, 1));
  LOOM_WAIT_LGKM0();
  barrier_nofence();          // (the state's loads stay in flight)
  for (int d0 = 0; d0 < D; d0 += N * NG) {
    if (d0 > 0) load(d0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = d0 + grp + NG * i;
      if (in && d < D) {
        const float k = s_k[d], q = s_q[d];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          x[i][y] = decayed_plus(x[i][y], a, k * v[y]);
          o[y] = __builtin_fmaf(q, x[i][y], o[y]);
        }
        store_stream(reinterpret_cast<f32x4_t*>(at + (int64_t)d * E), x[i]);
      }
    }
  }
  s_o[tid] = o;
  __syncthreads();
  if (grp == 0 && in) {
    for (int y = 1; y < NG; ++y) o += s_o[y * L + l];
    *reinterpret_cast<u32x2_t*>(p.out + bgh * E + e) =
        u32x2_t{pack2<F16>(o[0], o[1]), pack2<F16>(o[2], o[3])};
  }
}

// The launch's shape, from the extents alone.
struct Shape {
  int waves, nsl, nseg, cps;
};
Shape shape_of(int64_t B, int64_t G, int64_t H, int64_t D, int64_t E, int64_t T) {
  Shape s{};
  // 128 columns to a workgroup, 64 of states that are no wider
  s.waves = E <= 64 ? 4 : 8;
  s.nsl = (int)cdiv64(E, 16 * s.waves);
  const int64_t wgs = B * G * H * s.nsl, chunks = cdiv64(T, kC);
  // Segments of at least four chunks (T512 of 16 heads 20.0 us, of eight chunks 28.2, of two
  // 18.5; T2048 of 8 heads 26.9, 31.4, 37.9), as many workgroups as run at once.  More of
  // them cost more in the first launch than they balance (256 heads of prompts of 1024 to
  // 4096 cut in two 285 us, whole 197; 160 of T4096 in three 237, whole 193), and so did two
  // stretches to a segment for the first launch, whose states a segment's start adds up one
  // by one (T8192 of one head 110 us, 65 without; T512 of 16 20.4).
  // (Of eight waves two workgroups run on a CU too up to D 64 in bf16: not counted.)
  const int64_t slots = s.waves == 4 && D <= 128 ? 512 : 256;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>({slots / wgs, chunks / 4, 64}));
  s.cps = (int)cdiv64(chunks, want);
  s.nseg = (int)cdiv64(chunks, s.cps);
  return s;
}

template <bool F16, bool ONLY_STATE>
void launch_chunks(const LinearParams& p, const Shape& s, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.B * p.G * p.H * s.nsl *
                             (ONLY_STATE ? s.nseg - 1 : s.nseg))),
      block(64 * s.waves);
  auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, grid, block, 0, st, p); };
  // the kernel built for 64, 128 or 256 (the next one up) runs any narrower key dim
  if (s.waves == 4) {
    if (p.D > 128) launch(linear_chunk_kernel<256, 4, F16, ONLY_STATE>);
    else if (p.D > 64) launch(linear_chunk_kernel<128, 4, F16, ONLY_STATE>);
    else launch(linear_chunk_kernel<64, 4, F16, ONLY_STATE>);
  } else {
    if (p.D > 128) launch(linear_chunk_kernel<256, 8, F16, ONLY_STATE>);
    else if (p.D > 64) launch(linear_chunk_kernel<128, 8, F16, ONLY_STATE>);
    else launch(linear_chunk_kernel<64, 8, F16, ONLY_STATE>);
  }
}

template <bool F16, bool STEP>
int linear_impl(const void* q, const void* k, const void* v,
                const void* log_decay, const void* state, const void* counts, void* out,
                void* state_out, void* workspace, size_t workspace_bytes, int64_t B, int64_t G,
                int64_t H, int64_t D, int64_t E, int64_t T, float scale, void* stream, char* err,
                size_t errlen) {
  const char* const what = STEP ? "linear_attention_step" : "linear_attention";
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
  const size_t need = STEP ? 0 : loom_hip_linear_attention_workspace_bytes(B, G, H, D, E, T);
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
  if constexpr (STEP) {
    // 32 lanes of four columns to a row, fewer where there are few states
    int L = 32;
    while (L > 8 && (4 * (L / 2) >= E || B * G * H * cdiv64(E, 4 * L) < 512)) L /= 2;
    p.nsl = (int)cdiv64(E, 4 * L);
    hipLaunchKernelGGL((linear_step_kernel<F16>), dim3((unsigned)(B * G * H * p.nsl)), dim3(256), 0,
                       st, p, L);
    return loom_check_launch(err, errlen, what);
  }
  const Shape s = shape_of(B, G, H, D, E, T);
  p.ws = static_cast<float*>(workspace);
  p.nsl = s.nsl;
  p.nseg = s.nseg;
  p.cps = s.cps;
  if (s.nseg > 1) {
    launch_chunks<F16, true>(p, s, st);
    int rc = loom_check_launch(err, errlen, "linear_attention (states)");
    if (rc) return rc;
  }
  launch_chunks<F16, false>(p, s, st);
  return loom_check_launch(err, errlen, what);
}

}  // namespace

extern "C" {

size_t loom_hip_linear_attention_workspace_bytes(int64_t B, int64_t G, int64_t H, int64_t D,
                                                 int64_t E, int64_t T) {
  if (B <= 0 || G <= 0 || H <= 0 || D <= 0 || E <= 0 || T <= 0) return 0;
  // what does not fit is reported as no size at all fits
  if (T > (1 << 29) || D > 256 || E > 256 || !loom_prod_le({B, G, H}, 1 << 20)) return SIZE_MAX;
  const Shape s = shape_of(B, G, H, D, E, T);
  return s.nseg == 1 ? 0 : (size_t)(B * G * H * s.nseg) * D * E * 4;
}

int loom_hip_linear_attention(const void* q, const void* k, const void* v, const void* log_decay,
                              const void* state, const void* counts, void* out, void* state_out,
                              void* workspace, size_t workspace_bytes, int64_t B, int64_t G,
                              int64_t H, int64_t D, int64_t E, int64_t T, float scale,
                              void* stream, char* err, size_t errlen) {
  return linear_impl<false, false>(q, k, v, log_decay, state, counts, out, state_out,
                            workspace, workspace_bytes, B, G, H, D, E, T, scale, stream, err,
                            errlen);
}
int loom_hip_linear_attention_f16(const void* q, const void* k, const void* v,
                                  const void* log_decay, const void* state, const void* counts,
                                  void* out, void* state_out, void* workspace,
                                  size_t workspace_bytes, int64_t B, int64_t G, int64_t H,
                                  int64_t D, int64_t E, int64_t T, float scale, void* stream,
                                  char* err, size_t errlen) {
  return linear_impl<true, false>(q, k, v, log_decay, state, counts, out, state_out,
                           workspace, workspace_bytes, B, G, H, D, E, T, scale, stream, err,
                           errlen);
}

int loom_hip_linear_attention_step(const void* q, const void* k, const void* v,
                                   const void* log_decay, void* state, const void* counts,
                                   void* out, int64_t B, int64_t G, int64_t H, int64_t D,
                                   int64_t E, float scale, void* stream, char* err,
                                   size_t errlen) {
  return linear_impl<false, true>(q, k, v, log_decay, state, counts, out, state,
                            nullptr, 0, B, G, H, D, E, 1, scale, stream, err, errlen);
}
int loom_hip_linear_attention_step_f16(const void* q, const void* k, const void* v,
                                       const void* log_decay, void* state, const void* counts,
                                       void* out, int64_t B, int64_t G, int64_t H, int64_t D,
                                       int64_t E, float scale, void* stream, char* err,
                                       size_t errlen) {
  return linear_impl<true, true>(q, k, v, log_decay, state, counts, out, state,
                           nullptr, 0, B, G, H, D, E, 1, scale, stream, err, errlen);
}

}  // extern "C"
