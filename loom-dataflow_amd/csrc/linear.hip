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
#include <type_traits>

namespace {

constexpr int kC = 64;            // tokens of a chunk
constexpr int kIT = kC / 16, kM = kC / 32;

struct LinearParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const float* g;        // log decays
  const float* state;
  const int* counts;
  uint16_t* out;
  float* state_out;
  float* ws;             // [B G H, nseg, D, E]: what a segment starts from
  int B, G, H, D, E, T;
  int nsl;               // slices of E
  int nseg, cps;         // segments of a prompt, chunks to one
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

// A row's 16-byte chunks are XORed with this, so that both the 16 rows of a direct
// read (one chunk each) and the 8 consecutive rows of a transposed read's pass (a pair
// of chunks each) lie on distinct banks: rows of 128 bytes and of multiples of 256.
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
LOOM_DEV float finite_abs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }

// A value that the compiler does not know to be x: what rare paths compute from it is
// worked out there, not ahead of a loop in registers that it needs
LOOM_DEV int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The same address in every lane, stated to the compiler
LOOM_DEV const char* uniform(const char* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const char*>(
      ((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32) |
      (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v));
}

// Chunked form.  A workgroup of W waves walks the chunks of 64 tokens of one (b, g, h)
// and 16 W columns of E in order, each wave holding the state's D x 16 columns in the
// accumulators of its MFMAs, fp32.  For a chunk of tokens 0 .. C-1 and the state S before
// it:
//   P_ij = scale a^(i-j) q_i.k_j (j <= i),
//   out_i = sum_j P_ij v_j + scale a^(i+1) S^T q_i,
//   S' = a^C S + sum_j k_j (a^(C-1-j) v_j)^T.
// The MFMAs compute transposed tiles, S^T[e, d] . Q^T[d, i] and V^T[e, j] . P^T[j, i], so
// that a wave's state feeds the first product from its own accumulators (packed to 16
// bits: lane group g holds rows d = 16 t + 4 g + 0..3, and q's pieces are read in that
// order), and P^T is built from the accumulators of K Q^T, a part of it to each wave,
// shared through LDS.
// Rounding: S and P to 16 bits as operands, each once; a^(C-1-j) v_j as a sum of three
// bf16 or two f16 numbers, so that the state keeps fp32's accuracy.  f16 operands are
// scaled by powers of two where they leave its range.
// ONLY_STATE: a segment's own state from zero (the first's from the initial state), which
// later segments start from.
template <int DK, int W, bool F16, bool ONLY_STATE>
__global__ void __launch_bounds__(64 * W, 1) linear_chunk_kernel(LinearParams p) {
  constexpr int SL = 16 * W;                    // columns of a workgroup
  constexpr int KROW = DK * 2, VROW = SL * 2;
  constexpr int Q_BYTES = ONLY_STATE ? 0 : kC * KROW, K_BYTES = kC * KROW, V_BYTES = kC * VROW;
  constexpr int STAGE = Q_BYTES + K_BYTES + V_BYTES;
  constexpr int QK_INSTR = K_BYTES / 1024 / W, V_INSTR = V_BYTES / 1024 / W;
  static_assert(QK_INSTR >= 1 && V_INSTR >= 1, "every wave issues copies");
  constexpr int KS = DK / 32, DT = DK / 16;
  constexpr int MPW = W == 8 ? kM / 2 : kM;     // key pairs of the wave's part of P
  constexpr int TERMS = F16 ? 2 : 3;            // 16-bit numbers that hold a^(C-1-j) v_j
  static_assert(W == 4 || W == 8, "four query tiles");
  __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
  __shared__ __attribute__((aligned(16))) u32x4_t s_p[ONLY_STATE ? 1 : kIT * kM * 64];
  __shared__ float s_pow[kC + 1];
  __shared__ float s_ps[kIT * kM];              // f16: what a part of P was scaled by

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
  // a segment's own state is asked for by those behind it only
  const bool wanted = !ONLY_STATE || (seg + 1) * seglen < c;
  if (seg > 0 && (!wanted || t0 >= c)) return;
  const int tokens = wanted ? (int)min((int64_t)(c - t0), seglen) : 0;
  const int nch = (tokens + kC - 1) / kC;

  const float lg = p.g[gh];
  if (tid <= kC) s_pow[tid] = (float)decay_pow(lg, tid);
  // over a whole chunk, and over the last one
  const Decay full = split_decay(decay_pow(lg, kC));
  const Decay last = split_decay(decay_pow(lg, tokens - (nch - 1) * kC));

  // ---- copies of chunk ci into stage s: rows past the sequence and chunks past D or E
  // from zeros.  A whole chunk of whole rows takes each copy as the chunk's scalar base
  // plus this lane's offset, computed once (fast: all offsets fit 32 bits).
  const int64_t tok0 = (int64_t)b * p.T + t0;
  const uint16_t* const qb = p.q + (tok0 * GH + gh) * D;
  const uint16_t* const kb = p.k + (tok0 * p.G + g) * D;
  const uint16_t* const vb = p.v + (tok0 * p.G + g) * E + sl * SL;
  // token strides in bytes (at most 2^29)
  const uint32_t qs = (uint32_t)(GH * D * 2), ks_ = (uint32_t)(p.G * D * 2),
                 vs = (uint32_t)(p.G * E * 2);
  const bool fast = D == DK && sl * SL + SL <= E && qs < (1u << 25) && vs < (1u << 25);
  uint32_t qoff[QK_INSTR], koff[QK_INSTR], voff[V_INSTR];
  auto offsets = [&](auto& off, uint32_t stride, auto n) {
    constexpr int N = decltype(n)::value, INSTR = kC * N * 2 / 1024 / W;
#pragma unroll
    for (int i = 0; i < INSTR; ++i) {
      const int e = (wave * INSTR + i) * 64 + lane, row = e / (N / 8);
      off[i] = row * stride + ((e % (N / 8)) ^ row_swz<N>(row)) * 16;
    }
  };
  using QK = std::integral_constant<int, DK>;
  using VC = std::integral_constant<int, SL>;
  offsets(qoff, qs, QK{});
  offsets(koff, ks_, QK{});
  offsets(voff, vs, VC{});
  auto issue = [&](int s, int ci) {
    const int left = tokens - ci * kC;
    const uint32_t base = lds_addr((lds_char_t*)(smem + s * STAGE));
    auto rows = [&](const uint16_t* from, uint32_t stride, int valid, auto& off, auto n,
                    uint32_t lds) {
      constexpr int N = decltype(n)::value, INSTR = kC * N * 2 / 1024 / W;
      const char* at = uniform((const char*)from + (int64_t)ci * kC * stride);
      if (fast && left >= kC) {
#pragma unroll
        for (int i = 0; i < INSTR; ++i)
          dma_load16_s(off[i], at,
                       __builtin_amdgcn_readfirstlane(lds + (wave * INSTR + i) * 1024));
        return;
      }
      const int ln = fresh(lane);
#pragma unroll
      for (int i = 0; i < INSTR; ++i) {
        const int j = wave * INSTR + i;
        const int e = j * 64 + ln, row = e / (N / 8), ch = (e % (N / 8)) ^ row_swz<N>(row);
        const void* src = row < left && ch < valid
                              ? (const void*)(at + (int64_t)row * stride + ch * 16)
                              : (const void*)(loom_zero_kb + lane * 4);
        dma_load16(src, __builtin_amdgcn_readfirstlane(lds + j * 1024));
      }
    };
    if constexpr (!ONLY_STATE) rows(qb, qs, D / 8, qoff, QK{}, base);
    rows(kb, ks_, D / 8, koff, QK{}, base + Q_BYTES);
    rows(vb, vs, (E - sl * SL) / 8, voff, VC{}, base + Q_BYTES + K_BYTES);
  };
  if (nch > 0) issue(0, 0);

  // ---- the state: s[dt][i] is row d = 16 dt + 4 g4 + i, column ec
  const int col0 = sl * SL + wave * 16, ec = col0 + r;
  f32x4_t s[DT];
  const int64_t bgh = (int64_t)b * GH + gh, sz = (int64_t)D * E;
  // by buffer accesses, which the hardware checks against the state's end: rows past D
  // and columns past E read as zeros and are not written
  const uint32_t sbytes = (uint32_t)(D * E * 4);
  const uint32_t sbase = ec < E ? (uint32_t)(4 * g4 * E + ec) * 4 : 1u << 30;
  auto read_state = [&](const float* from, f32x4_t (&x)[DT]) {
    const rsrc_t rs = make_rsrc(from, sbytes);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[dt][i] = __uint_as_float(buf_load4(rs, sbase + (uint32_t)((16 * dt + i) * E) * 4));
  };
  auto write_state = [&](float* to) {
    const rsrc_t rs = make_rsrc(to, sbytes);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s[dt][i]), rs,
                                              sbase + (uint32_t)((16 * dt + i) * E) * 4, 0, 0);
  };
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) s[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (p.nseg == 1 || (ONLY_STATE && seg == 0)) {
    if (p.state) read_state(p.state + bgh * sz, s);
    // (state_out may be state: the first segment reads a copy)
    if constexpr (ONLY_STATE) write_state(p.ws + bgh * p.nseg * sz);
  } else if constexpr (!ONLY_STATE) {
#pragma unroll 1
    for (int u = seg == 0 ? 0 : 1; u <= seg; ++u) {
      const float w = (float)exp((double)(seg - u) * (double)seglen *
                                 (double)(lg < -1e30f ? -1e30f : lg));
      f32x4_t x[DT];
      read_state(p.ws + (bgh * p.nseg + u) * sz, x);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) s[dt] += x[dt] * w;
    }
  }

  // ---- factors, the same for every whole chunk
  __syncthreads();          // (s_pow)
  float w[kM][8], rise[kIT];
#pragma unroll
  for (int m = 0; m < kM; ++m)
#pragma unroll
    for (int x = 0; x < 8; ++x) w[m][x] = s_pow[kC - 1 - (32 * m + 16 * (x >> 2) + 4 * g4 + (x & 3))];
#pragma unroll
  for (int it = 0; it < kIT; ++it) rise[it] = p.scale * s_pow[16 * it + r + 1];
  // this wave's part of P: queries 16 pit .., key pairs pm0 .. pm0 + MPW - 1
  const int pit = wave & 3, pm0 = W == 8 ? wave >> 2 : 0;
  float pf_fac[2 * MPW][4];
#pragma unroll
  for (int t = 0; t < 2 * MPW; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int lag = 16 * pit + r - (16 * (2 * pm0 + t) + 4 * g4 + e);
      pf_fac[t][e] = lag >= 0 ? p.scale * s_pow[lag] : -1.f;    // -1: not seen
    }
  const bool stores = !ONLY_STATE && col0 < E;
  const char* const ob = reinterpret_cast<const char*>(p.out + (tok0 * GH + gh) * E + col0);
  const int64_t ooff = (int64_t)r * GH * E * 2 + 8 * g4;
  // stores of a chunk's rows, all of which a whole chunk issues
  constexpr int STORES = kIT;

  for (int ci = 0; ci < nch; ++ci) {
    char* const st = smem + (ci & 1) * STAGE;
    lds_char_t* const lq = (lds_char_t*)st;
    lds_char_t* const lk = (lds_char_t*)(st + Q_BYTES);
    lds_char_t* const lv = (lds_char_t*)(st + Q_BYTES + K_BYTES);
    const int left = tokens - ci * kC;
    lds_order();
    // the copies of this chunk; the stores of the one before are younger
    if (stores && ci > 0) LOOM_WAIT_VMCNT(STORES);
    else LOOM_WAIT_VMCNT(0);
    LOOM_WAIT_LGKM0();
    barrier_nofence();
    if (ci + 1 < nch) issue(~ci & 1, ci + 1);

    // rows 16 t + r of q or k, elements d = 32 ks + 4 g4 .. and 32 ks + 16 + 4 g4 ..
    auto row_op = [&](const lds_char_t* base, int t, int ks) {
      const int row = 16 * t + r, sw = row_swz<DK>(row);
      const lds_char_t* at = base + row * KROW + (g4 & 1) * 8;
      typedef __attribute__((address_space(3))) u32x2_t lds_u32x2;
      const u32x2_t lo = *reinterpret_cast<const lds_u32x2*>(at + ((4 * ks + (g4 >> 1)) ^ sw) * 16);
      const u32x2_t hi =
          *reinterpret_cast<const lds_u32x2*>(at + ((4 * ks + 2 + (g4 >> 1)) ^ sw) * 16);
      return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
    };
    // column tile x of K^T or V^T, tokens 32 m + 4 g4 .. and 32 m + 16 + 4 g4 ..
    auto col_op = [&](const lds_char_t* base, auto n, int m, int x) {
      constexpr int N = decltype(n)::value;
      const int row = 32 * m + 4 * g4 + a4;
      const lds_char_t* at =
          base + row * (N * 2) + ((2 * x + (c4 >> 1)) ^ row_swz<N>(row)) * 16 + (c4 & 1) * 8;
      const u32x2_t lo = lds_read_tr16(at);
      const u32x2_t hi = lds_read_tr16(at + 16 * (N * 2));    // (the same swizzle)
      return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
    };

    if constexpr (!ONLY_STATE) {
      // ---- this wave's part of P^T, as the operands that every wave reads
      u32x4_t qf[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = row_op(lq, pit, ks);
#pragma unroll
      for (int mm = 0; mm < MPW; ++mm) {
        const int m = pm0 + mm;
        if (2 * m > pit) continue;              // wave-uniform
        f32x4_t x[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          x[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
          if (2 * m + t <= pit) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
              x[t] = mfma16t<F16>(row_op(lk, 2 * m + t, ks), qf[ks], x[t]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = pf_fac[2 * mm + t][e];
            x[t][e] = f >= 0.f ? x[t][e] * f : 0.f;
          }
        }
        if constexpr (F16) {
          float mx = 0.f;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, finite_abs(x[t][e]));
          const float sc = f16_scale(mx);
#pragma unroll
          for (int t = 0; t < 2; ++t) x[t] *= sc;
          if (lane == 0) s_ps[pit * kM + m] = sc;
        }
        s_p[(pit * kM + m) * 64 + lane] =
            u32x4_t{pack2<F16>(x[0][0], x[0][1]), pack2<F16>(x[0][2], x[0][3]),
                    pack2<F16>(x[1][0], x[1][1]), pack2<F16>(x[1][2], x[1][3])};
      }
    }

    __builtin_amdgcn_sched_barrier(0);
    // ---- S^T Q^T of the state before the chunk, times scale a^(i+1)
    f32x4_t o[kIT];
    if constexpr (!ONLY_STATE) {
      float sc = 1.f;
      if constexpr (F16) {
        float mx = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, finite_abs(s[dt][i]));
        sc = f16_scale(mx);
      }
      u32x4_t sp[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        f32x4_t x = s[2 * ks], y = s[2 * ks + 1];
        if constexpr (F16) {
          x *= sc;
          y *= sc;
        }
        sp[ks] = u32x4_t{pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]), pack2<F16>(y[0], y[1]),
                         pack2<F16>(y[2], y[3])};
      }
      const float back = F16 ? 1.f / sc : 1.f;
#pragma unroll
      for (int it = 0; it < kIT; ++it) {
        o[it] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) o[it] = mfma16t<F16>(sp[ks], row_op(lq, it, ks), o[it]);
        o[it] *= rise[it] * back;
        // (two tiles' reads at a time: all at once would not leave registers enough)
        if (it & 1) __builtin_amdgcn_sched_barrier(0);
      }
    }

    __builtin_amdgcn_sched_barrier(0);
    // ---- the state behind the chunk
    u32x4_t vf[kM], vt[TERMS][kM];
#pragma unroll
    for (int m = 0; m < kM; ++m) vf[m] = col_op(lv, VC{}, m, wave);
    Decay a = full;
    if (left < kC) {          // the last, partial chunk
      a = last;
      const int j0 = fresh(4 * g4);
#pragma unroll
      for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int x = 0; x < 8; ++x)
          w[m][x] = s_pow[max(0, left - 1 - (32 * m + 16 * (x >> 2) + j0 + (x & 3)))];
    }
    // f16: the second number 2^11 times larger, in sums of its own, so that it keeps
    // its bits
    constexpr float kLow = F16 ? 2048.f : 1.f;
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float y0 = lo16<F16>(vf[m][x]) * w[m][2 * x], y1 = hi16<F16>(vf[m][x]) * w[m][2 * x + 1];
#pragma unroll
        for (int z = 0; z < TERMS; ++z) {
          const uint32_t y = pack2<F16>(y0, y1);
          vt[z][m][x] = y;
          if (z + 1 < TERMS) {
            y0 = (y0 - lo16<F16>(y)) * kLow;
            y1 = (y1 - hi16<F16>(y)) * kLow;
          }
        }
      }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      f32x4_t x = f32x4_t{0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll
      for (int m = 0; m < kM; ++m) {
        const u32x4_t kt = col_op(lk, QK{}, m, dt);
        if constexpr (F16) {
          x = mfma16t<F16>(kt, vt[0][m], x);
          y = mfma16t<F16>(kt, vt[1][m], y);
        } else {              // (the small ones in sums of their own: half the chain)
          x = mfma16t<F16>(kt, vt[0][m], x);
          y = mfma16t<F16>(kt, vt[TERMS - 1][m], y);
          y = mfma16t<F16>(kt, vt[1][m], y);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float z = F16 ? __builtin_fmaf(y[i], 1.f / kLow, x[i]) : x[i] + y[i];
        s[dt][i] = __builtin_fmaf(s[dt][i], a.hi, __builtin_fmaf(s[dt][i], a.lo, z));
      }
      if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }

    if constexpr (!ONLY_STATE) {
      __builtin_amdgcn_sched_barrier(0);
      // ---- V^T P^T of the chunk's own tokens
      // A token whose v is not finite makes its columns of the state so: then every
      // query takes its own product, tokens behind it as zeros, since a weight of zero
      // times an infinity would reach the queries ahead of them.
      const bool alone = __builtin_amdgcn_ballot_w64(!(fabsf(s[0][0]) < INFINITY)) != 0;
      LOOM_WAIT_LGKM0();
      barrier_nofence();
#pragma unroll
      for (int it = 0; it < kIT; ++it) {
#pragma unroll
        for (int m = 0; m <= it / 2; ++m) {
          const u32x4_t pf = s_p[(it * kM + m) * 64 + lane];
          float ps = 1.f;
          if constexpr (F16) {
            ps = s_ps[it * kM + m];
            o[it] *= ps;
          }
          if (!alone || 32 * m + 31 <= 16 * it) {
            o[it] = mfma16t<F16>(vf[m], pf, o[it]);
          } else {
            const int j0 = fresh(4 * g4);
#pragma unroll 1
            for (int x = 0; x < 16; ++x) {
              u32x4_t keep;
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const int j = 32 * m + 16 * (y >> 1) + j0 + 2 * (y & 1), i = 16 * it + x;
                keep[y] = (j <= i ? 0xffffu : 0u) | (j + 1 <= i ? 0xffff0000u : 0u);
              }
              const f32x4_t z = mfma16t<F16>(vf[m] & keep, pf, o[it]);
              if (r == x) o[it] = z;
            }
          }
          if constexpr (F16) o[it] *= 1.f / ps;
        }
        // ---- o[it][e] is token 16 it + r, column col0 + 4 g4 + e
        const char* to = uniform(ob + (int64_t)(ci * kC + 16 * it) * GH * E * 2);
        if (16 * it + r < left && col0 + 4 * g4 < E)
          *reinterpret_cast<u32x2_t*>(const_cast<char*>(to) + ooff) =
              u32x2_t{pack2<F16>(o[it][0], o[it][1]), pack2<F16>(o[it][2], o[it][3])};
      }
    }
  }

  if constexpr (ONLY_STATE) {
    if (!wanted) return;
    write_state(p.ws + (bgh * p.nseg + seg + 1) * sz);
  } else if (t0 + tokens == c) {      // the segment that the sequence ends in
    write_state(p.state_out + bgh * sz);
  }
}

// One token.  L lanes of four columns to a row of the state, 256 / L rows at once.
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
          x[i][y] = __builtin_fmaf(x[i][y], a.hi, __builtin_fmaf(x[i][y], a.lo, k * v[y]));
          o[y] = __builtin_fmaf(q, x[i][y], o[y]);
        }
        *reinterpret_cast<f32x4_t*>(at + (int64_t)d * E) = x[i];
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
  // 128 columns to a workgroup; 64 of states that are no wider, and past D 128, where the
  // stages of 128 do not fit
  s.waves = D > 128 || E <= 64 ? 4 : 8;
  s.nsl = (int)cdiv64(E, 16 * s.waves);
  const int64_t wgs = B * G * H * s.nsl, chunks = cdiv64(T, kC);
  // workgroups that run at once
  const int64_t slots = D > 64 ? 256 : 512;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>({slots / wgs, chunks / 4, 64}));
  s.cps = (int)cdiv64(chunks, want);
  s.nseg = (int)cdiv64(chunks, s.cps);
  return s;
}

template <bool F16, bool ONLY_STATE>
void launch_chunks(const LinearParams& p, const Shape& s, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.B * p.G * p.H * s.nsl * (s.nseg - (ONLY_STATE ? 1 : 0)))),
      block(64 * s.waves);
  auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, grid, block, 0, st, p); };
  // the kernel built for 64, 128 or 256 (the next one up) runs any narrower key dim
  if (p.D > 128) launch(linear_chunk_kernel<256, 4, F16, ONLY_STATE>);
  else if (p.D > 64) {
    if (s.waves == 4) launch(linear_chunk_kernel<128, 4, F16, ONLY_STATE>);
    else launch(linear_chunk_kernel<128, 8, F16, ONLY_STATE>);
  } else {
    if (s.waves == 4) launch(linear_chunk_kernel<64, 4, F16, ONLY_STATE>);
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
