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
//
// gfx950 mapping.  The own keys are bound by streaming K and V once (H heads
// give H operations a byte); the prefix, whose K and V all B H rows of a head
// share, by the matrix cores or, in short calls, by latency.  Two launches:
//   - cache_split_kernel: every workgroup takes a *part*, some query rows
//     against a range of keys of one K, V, and leaves (base, sum, sum of p v):
//     parts of the prefix (tiles of 32, 64 or 128 of the B H rows, key splits)
//     and chunks of each sequence's own keys.  They run side by side, so that the
//     prefix's arithmetic hides behind the caches' stream (B48 G8 H8 P16384 S4096:
//     prefix alone 51 us, own keys alone 98, together 113);
//   - cache_join_kernel: joins a row's parts and, from the scores that the chunks
//     left in the workspace, adds the weights.  Scores are kept in fp32: weights
//     are sums of many steps.  Written and read they are 8 H bytes a key, a second
//     reading of K 2 D: as many at 32 heads of D 128, and fewer scores below.  Above
//     that (71 heads of D 64: 568 bytes against 128) K would be the smaller; no
//     kernel here scores it twice, and what that would take is not measured.
// Rounding: scores, bases and sums are fp32; p is rounded to 16 bits for its
// product with v, and out is divided by the sum of the rounded p, so that one
// heavy key's rounding cancels.  The weights use the unrounded p and their own sum.
// f16 rounds below 2^-14 to multiples of 2^-24, so its p are held 2^7 times larger
// (the base lies that far below the largest score): a key down to 2^-21 of the heaviest
// of its part keeps all eleven bits, one below 2^-32 is lost, as below 2^-25 without.
#include "common.h"

#include <climits>
#include <cmath>
#include <type_traits>

namespace {

constexpr int kThreads = 256;     // four waves
constexpr int kKeys = 64;         // keys per stage

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
  int2* plan;       // [B]: a sequence's first chunk and their number
  f32x4_t* ml;      // per partial row: base, sum of p, sum of the rounded p
  float* o;         // per partial row: sum of p v, D values
  float* score;     // [B G, H, Sp] scores of the own keys, log2 domain
  int B, G, H, D, P, S, Sp;
  int nht;          // row tiles of a (b, g)'s H heads
  int chunks;       // chunks that the whole batch aims at
  int most;         // chunks that it has at most
  int rtp, ntp, nsp, tile_p;   // the prefix: rows of a tile, tiles per head, splits, keys of one
  int nprefix;      // workgroups of the prefix
  int njoin, flat;  // workgroups that join rows; several rows to each
  int once;         // own keys are read by non-temporal copies
  int wkeys;        // keys of a workgroup that gathers weights: 128 to 1024
  float c2;         // scale * log2(e)
};

LOOM_DEV int seq_len(const StepParams& p, int b) { return min(max(p.lens[b], 0), p.S); }

// ---------------------------------------------------------------------------
// One part: up to RT query rows against the keys [s0, s1) of one K, V.
// ---------------------------------------------------------------------------
// Own keys of caches larger than the 256 MB last-level cache are copied by
// dma_once16, so that the stream displaces nothing that is read again (B48 G8 S4096 under a prefix 124 -> 113 us a step, B8 G8
// S8192 43.5 -> 38.7); smaller ones may still lie there from the last step (B16
// G8 S2048 29.3 against 31.6), and a prefix is read by many sequences.  The rule
// knows the capacity, not the lengths: large caches that hold little pay up to 5%
// (B48 G8 H8 S8192 holding 1024 to 1536 keys each 55.6 against 53.1 us, 100 to 400
// keys 20.6 against 20.0).
struct Part {
  const uint16_t* k;    // [D][ld]
  const uint16_t* v;    // [ld][D]
  int ld;               // keys of a K row
  int s0, s1;           // this part's keys, s0 a multiple of 64
  int rows;             // query rows
  bool once;            // no other workgroup reads these keys
  int i0;               // first row: of the (b, g)'s heads, or of head g's B H rows
  int g;                // the KV head of a prefix part, -1: rows are consecutive
  int64_t out0;         // partial row of row 0; the others follow
  float* score;         // scores of row 0, Sp apart, or null
};

// Row lr of a part in q's [B G H] rows.  A prefix's rows are all sequences'
// heads of its g.
LOOM_DEV int64_t part_row(const StepParams& p, const Part& a, int lr) {
  const int i = a.i0 + lr;
  if (a.g < 0 || p.G == 1) return i;
  const int b = i / p.H;
  return ((int64_t)b * p.G + a.g) * p.H + (i - b * p.H);
}

// Four waves, 64 keys a stage, two stages (64 KB up to D 128, so two workgroups
// fit a CU and one's arithmetic covers the other's waits).  As in
// decode.hip: K [d][key] and V [key][d] lie in LDS as the tensors have them,
// copied by LDS DMA (K through registers where its rows start off 16-byte
// boundaries, KREG), and reach the MFMAs by transposed reads,
//   S^T[key, row] = K^T . Q^T,   O^T[d, row] += V^T . P^T.
// KG 2: two waves share 16 QT rows, each taking one 32-key half of every stage,
// and merge at the end: 32 rows, for the heads of one KV head.  KG 1: a wave takes
// 16 QT rows of its own: 64 or 128 rows that share the stages.  WT: the scores
// of own keys are stored and the unrounded p summed.
template <int D, bool F16, bool WT, int QT, int KG, bool KREG>
LOOM_DEV void run_part(const StepParams& p, const Part& a, char* smem) {
  constexpr int W = kThreads / 64;
  constexpr int RT = 16 * QT * W / KG;          // rows of a workgroup
  constexpr int K_BYTES = D * kKeys * 2, V_BYTES = kKeys * D * 2;
  constexpr int STAGE = K_BYTES + V_BYTES;
  constexpr int K_INSTR = K_BYTES / 1024 / W, V_INSTR = V_BYTES / 1024 / W;
  constexpr int VROW = D * 2, V_ROWS_PER_I = 1024 / VROW;
  constexpr int DSTEPS = D / 32, DT = D / 16;
  constexpr int Q_INSTR = RT * D * 2 / 1024 / W;
  static_assert(RT * D * 2 <= STAGE, "the queries arrive in the second stage");

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int a4 = r >> 2, c4 = r & 3;            // transposed-read lane roles
  const int qw = wave / KG, kh = wave % KG;     // query rows and key half of this wave
  const int Dr = p.D, ld = a.ld, s0 = a.s0, s1 = a.s1;
  const uint16_t* __restrict__ kg = a.k;
  const uint16_t* __restrict__ vg = a.v;
  const int nblk = (s1 - s0 + kKeys - 1) / kKeys;
  const bool once = __builtin_amdgcn_readfirstlane((int)a.once) != 0;
  const bool active = 16 * QT * qw < a.rows;    // this wave has rows
  // score stores of a block that every active wave issues at least (those of
  // its first row tile): younger than the next block's copies, so the wait for
  // the copies need not wait for them
  const bool stores = WT && active && a.score;
  constexpr int STORES = KG == 2 ? 2 : 4;

  auto stK = [&](int s) { return (lds_char_t*)(smem + s * STAGE); };
  auto stV = [&](int s) { return (lds_char_t*)(smem + s * STAGE + K_BYTES); };
  // ---- DMA of block `blk` into stage s: K pieces past the row's end are
  // clamped (their keys are masked), rows d >= Dr come from zeros, and so do V
  // rows past s1 (slots behind a length may hold anything, and a weight of zero
  // times NaN or infinity is NaN)
  auto copies = [&](int s, int blk, auto once) {
    auto copy = [](const void* from, uint32_t to) {
      to = __builtin_amdgcn_readfirstlane(to);
      if constexpr (decltype(once)::value) dma_once16(from, to);
      else dma_load16(from, to);
    };
    const int kv0 = s0 + blk * kKeys;
    const uint32_t lk = lds_addr(stK(s)), lv = lds_addr(stV(s));
    if constexpr (!KREG) {
#pragma unroll
      for (int i = 0; i < K_INSTR; ++i) {
        const int j = wave * K_INSTR + i;
        const int d = j * 8 + lane / 8;
        const int key = min(kv0 + ((lane % 8) ^ k_swz(d)) * 8, ld - 8);
        if (j * 8 < Dr)                                 // wave-uniform
          copy(kg + (int64_t)d * ld + key, lk + j * 1024);
        else
          dma_load16(loom_zero_kb + lane * 4, __builtin_amdgcn_readfirstlane(lk + j * 1024));
      }
    }
#pragma unroll
    for (int i = 0; i < V_INSTR; ++i) {
      const int j = wave * V_INSTR + i;
      const int kr = j * V_ROWS_PER_I + lane / (D / 8);
      const int c = min((lane % (D / 8)) ^ v_swz<D>(kr), Dr / 8 - 1);
      const int key = kv0 + kr;
      const void* const from = key < s1 ? (const void*)(vg + (int64_t)key * Dr + c * 8)
                                        : (const void*)(loom_zero_kb + lane * 4);
      copy(from, lv + j * 1024);
    }
  };
  auto issue = [&](int s, int blk) {
    if (once) copies(s, blk, std::true_type{});
    else copies(s, blk, std::false_type{});
  };
  // ---- KREG (ld not a multiple of 8): K pieces through registers
  const rsrc_t krs = make_rsrc(kg, KREG ? (uint32_t)(Dr * ld * 2) : 0u);
  u32x4_t kr[KREG ? K_INSTR : 1];
  auto kload = [&](int blk) {
    const int kv0 = s0 + blk * kKeys;
#pragma unroll
    for (int i = 0; i < K_INSTR; ++i) {
      const int j = wave * K_INSTR + i;
      const int d = j * 8 + lane / 8;
      kr[i] = j * 8 < Dr ? row_piece8(krs, ld, d, kv0 + ((lane % 8) ^ k_swz(d)) * 8)
                         : u32x4_t{0u, 0u, 0u, 0u};
    }
  };
  auto kstore = [&](int s) {
#pragma unroll
    for (int i = 0; i < K_INSTR; ++i)
      *reinterpret_cast<__attribute__((address_space(3))) u32x4_t*>(
          stK(s) + (wave * K_INSTR + i) * 1024 + lane * 16) = kr[i];
  };

  // ---- the queries into the second stage (rows past the part's repeat its
  // last, elements past Dr are zeroed when read), then the first block
  lds_char_t* const sq = stK(1);
  // (a rolled loop: code that a workgroup runs once is fetched as it runs)
#pragma unroll 1
  for (int i = 0; i < Q_INSTR; ++i) {
    const int j = wave * Q_INSTR + i;
    const int e = j * 512 + lane * 8;
    const int64_t row = part_row(p, a, min(e / D, a.rows - 1));
    dma_load16(p.q + row * Dr + min(e % D, Dr - 8), lds_addr(sq) + j * 1024);
  }
  issue(0, 0);
  if constexpr (KREG) {     // (its wait covers V's copies, on their way before it)
    kload(0);
    kstore(0);
  }

  u32x4_t qf[DSTEPS][QT];
  const float c2 = p.c2;
  // log2 of what the largest p starts at, and how far it may rise: to 2^15, half of
  // f16's largest number (bf16 has fp32's exponents)
  constexpr float kLift = F16 ? 7.f : 0.f, kRise = kLift + 8.f;
  float m_run[QT], lx[QT];
  f32x4_t ot[DT][QT], lacc[QT];
  const u32x4_t ones = u32x4_t{kOnePair<F16>, kOnePair<F16>, kOnePair<F16>, kOnePair<F16>};
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m_run[qt] = lx[qt] = 0.f;
    lacc[qt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) ot[dt][qt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  bool first = true;

  // ---- this wave's keys of block blk in stage s (one 32-key half with two key
  // groups, else both) against its rows
  constexpr int NH = 2 / KG;
  auto compute = [&](int s, int blk) {
    const int kv0 = s0 + blk * kKeys + 32 * (KG == 2 ? kh : 0);
    const lds_char_t* ks = stK(s);
    const lds_char_t* vs = stV(s);
    // K^T operand of 16 keys jt, 32 d; V^T operand of 16 d, 32 keys hv.  A half's
    // are read well before the MFMAs that use them, V's before the softmax:
    // left to itself the compiler keeps two in flight, and every MFMA waits
    // for the LDS
    auto k_op = [&](int jt, int ds) {
      const int d = ds * 32 + g * 8 + a4;
      const int ch = (2 * jt + (c4 >> 1)) ^ k_swz(d);
      const lds_char_t* q = ks + d * (kKeys * 2) + ch * 16 + (c4 & 1) * 8;
      const u32x2_t lo = lds_read_tr16(q);
      const u32x2_t hi = lds_read_tr16(q + 4 * (kKeys * 2));
      return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
    };
    auto v_op = [&](int hv, int dt) {
      const int k0r = 32 * hv + 4 * g + a4;
      const int ch = (2 * dt + (c4 >> 1)) ^ v_swz<D>(k0r);
      const lds_char_t* q = vs + k0r * VROW + ch * 16 + (c4 & 1) * 8;
      const u32x2_t lo = lds_read_tr16(q);
      const u32x2_t hi = lds_read_tr16(q + 16 * VROW);
      return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
    };
    constexpr int kFence = 0x0006;              // VALU and SALU may cross
    const int h0 = KG == 2 ? kh : 0;
    // st[j][qt][i]: key kv0 + 16 j + 4 g + i, row 16 qt + r of this wave
    f32x4_t st[2 * NH][QT];
#pragma unroll
    for (int j = 0; j < 2 * NH; ++j)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) st[j][qt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    u32x4_t kf[2][DSTEPS], vf[DT];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
#pragma unroll
      for (int ds = 0; ds < DSTEPS; ++ds)
#pragma unroll
        for (int j = 0; j < 2; ++j) kf[j][ds] = k_op(2 * (h0 + h) + j, ds);
      __builtin_amdgcn_sched_barrier(kFence);
#pragma unroll
      for (int ds = 0; ds < DSTEPS; ++ds)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            st[2 * h + j][qt] = mfma16t<F16>(kf[j][ds], qf[ds][qt], st[2 * h + j][qt]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vf[dt] = v_op(h0, dt);
    __builtin_amdgcn_sched_barrier(kFence);
    const bool edge = kv0 + 32 * NH > s1;
    if constexpr (WT) {
      if (a.score) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          const int lr = 16 * (QT * qw + qt) + r;
          float* to = a.score + (int64_t)lr * p.Sp + kv0 + 4 * g;
          if (lr < a.rows)
#pragma unroll
            for (int j = 0; j < 2 * NH; ++j)
              *reinterpret_cast<f32x4_t*>(to + 16 * j) = st[j][qt] * c2;
        }
      }
    }
    // log2-domain scores relative to the base; keys past s1 are -inf
    float lmax[QT];
    bool big = false;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2 * NH; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = __builtin_fmaf(st[j][qt][i], c2, -m_run[qt]);
          if (edge && kv0 + 16 * j + 4 * g + i >= s1) v = -INFINITY;
          st[j][qt][i] = v;
          mx = fmaxf(mx, v);
        }
      lmax[qt] = mx;
      big |= mx > kRise;
    }
    // lazy online softmax: a row's base is set by its first block with a
    // finite score and moves (O and the sums rescale) when one rises 2^8 above
    // that block's largest
    if (first || __builtin_amdgcn_ballot_w64(big) != 0) {
      bool unset_left = false;
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        float mx = lmax[qt];
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const bool unset = first && lacc[qt][0] == 0.f;
        const float shift = unset ? (mx == -INFINITY ? 0.f : mx - kLift) : fmaxf(mx - kLift, 0.f);
        const float alpha = unset ? 1.f : fast_exp2(-shift);
        lacc[qt] *= alpha;
        lx[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) ot[dt][qt] *= alpha;
        m_run[qt] += shift;
#pragma unroll
        for (int j = 0; j < 2 * NH; ++j) st[j][qt] -= shift;
        unset_left |= unset && mx == -INFINITY;
      }
      first = __builtin_amdgcn_ballot_w64(unset_left) != 0;
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      u32x4_t pf[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        f32x4_t e0, e1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e0[i] = fast_exp2(st[2 * h][qt][i]);
          e1[i] = fast_exp2(st[2 * h + 1][qt][i]);
        }
        if constexpr (WT)
          lx[qt] += ((e0[0] + e0[1]) + (e0[2] + e0[3])) + ((e1[0] + e1[1]) + (e1[2] + e1[3]));
        pf[qt] = u32x4_t{pack2<F16>(e0[0], e0[1]), pack2<F16>(e0[2], e0[3]),
                         pack2<F16>(e1[0], e1[1]), pack2<F16>(e1[2], e1[3])};
        lacc[qt] = mfma16t<F16>(ones, pf[qt], lacc[qt]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) ot[dt][qt] = mfma16t<F16>(vf[dt], pf[qt], ot[dt][qt]);
        if (h + 1 < NH) vf[dt] = v_op(h + 1, dt);
      }
    }
  };

  for (int it = 0; it < nblk; ++it) {
    const int s = it & 1;
    lds_order();
    if (it > 0 && stores) LOOM_WAIT_VMCNT(STORES);
    else LOOM_WAIT_VMCNT(0);
    LOOM_WAIT_LGKM0();
    barrier_nofence();
    if (it == 0) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int ds = 0; ds < DSTEPS; ++ds) {
          const int lr = 16 * (QT * qw + qt) + r;
          const u32x4_t raw = *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(
              sq + (lr * D + ds * 32 + g * 8) * 2);
          qf[ds][qt] = ds * 32 + g * 8 < Dr ? raw : u32x4_t{0u, 0u, 0u, 0u};
        }
      LOOM_WAIT_LGKM0();      // the second stage is overwritten next
      barrier_nofence();
    }
    const bool ahead = it + 1 < nblk;
    if constexpr (KREG) {
      if (ahead) kload(it + 1);
    }
    if (ahead) issue(s ^ 1, it + 1);
    if (active) compute(s, it);
    if constexpr (KREG) {
      if (ahead) kstore(s ^ 1);
    }
  }

  // ---- the sums of the four lane groups, each of which held other keys
  if constexpr (WT) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      lx[qt] += __shfl_xor(lx[qt], 16);
      lx[qt] += __shfl_xor(lx[qt], 32);
    }
  }
  // ---- KG 2: the pair's second wave hands its state over through the idle
  // stages, lane by lane (both hold the same rows and columns); a half without
  // a key of finite score (l = 0) takes no part
  if constexpr (KG == 2) {
    constexpr int SLOT = QT * (DT + 1) * 64;
    static_assert(W / 2 * SLOT * 16 <= 2 * STAGE, "merge area");
    LOOM_WAIT_LGKM0();
    barrier_nofence();
    f32x4_t* const mg = reinterpret_cast<f32x4_t*>(smem) + qw * SLOT + lane;
    if (kh == 1) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) mg[(qt * (DT + 1) + dt) * 64] = ot[dt][qt];
        mg[(qt * (DT + 1) + DT) * 64] = f32x4_t{lacc[qt][0], m_run[qt], lx[qt], 0.f};
      }
    }
    LOOM_WAIT_LGKM0();
    barrier_nofence();
    if (kh == 1) return;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const f32x4_t lm = mg[(qt * (DT + 1) + DT) * 64];
      const float l0 = lacc[qt][0], l1 = lm[0], m0 = m_run[qt], m1 = lm[1];
      const float M = l0 != 0.f ? (l1 != 0.f ? fmaxf(m0, m1) : m0) : m1;
      const float f0 = l0 != 0.f ? fast_exp2(m0 - M) : 0.f;
      const float f1 = l1 != 0.f ? fast_exp2(m1 - M) : 0.f;
      lacc[qt][0] = l0 * f0 + l1 * f1;
      lx[qt] = lx[qt] * f0 + lm[2] * f1;
      m_run[qt] = M;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        ot[dt][qt] = ot[dt][qt] * f0 + mg[(qt * (DT + 1) + dt) * 64] * f1;
    }
  }
  // ---- (base, sums, O) of every row.  ot[dt][qt][i] is d = 16 dt + 4 g + i of
  // row 16 qt + r: turned through this wave's stretch of the idle stages (16 rows
  // of D + 4 floats, free of conflicts) into whole rows, 16 bytes a lane.  Rolled
  // loops: a workgroup runs this once, and fetching unrolled code took longer
  // than the stores
  constexpr int OROW = D + 4, PPR = D / 4;      // floats and 16-byte pieces of a row
  constexpr int OFF = KG == 2 ? W / 2 * QT * (DT + 1) * 64 * 4 : 0;   // past the handed-over state
  static_assert(OFF * 4 + W / KG * 16 * OROW * 4 <= 2 * STAGE, "O rows fit the stages");
  if (KG == 1) {
    LOOM_WAIT_LGKM0();
    barrier_nofence();
  }
  float* const mo = reinterpret_cast<float*>(smem) + OFF + qw * 16 * OROW;
  const int lr0 = lane / PPR, c = (lane % PPR) * 4;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int t0 = 16 * (QT * qw + qt);         // first row of the tile
    const int n = min(16, a.rows - t0);
    const int64_t row0 = a.out0 + t0;
    if (r < n && g == 0) p.ml[row0 + r] = f32x4_t{m_run[qt], lx[qt], lacc[qt][0], 0.f};
    lds_order();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<f32x4_t*>(mo + r * OROW + dt * 16 + 4 * g) = ot[dt][qt];
    lds_order();
    if (c < Dr) {
      float* to = p.o + (row0 + lr0) * Dr + c;
#pragma unroll 1
      for (int lr = lr0; lr < n; lr += 64 / PPR, to += 64 / PPR * Dr)
        store_stream(reinterpret_cast<f32x4_t*>(to),
                     *reinterpret_cast<const f32x4_t*>(mo + lr * OROW + c));
    }
    lds_order();
  }
}

// Where chunk c of the batch's own keys lies.  t, a multiple of 64, is the chunk
// that gives about p.chunks of them over all sequences whatever their lengths,
// at least 128 keys (64 leave more parts to join than they save: B1 S16384 with
// weights 25.8 against 18.8 us a step, B32 of 256 to 1024 keys 16.0 and 13.7), and
// larger while that gives more than p.most of them; a sequence takes as many as t
// asks for, of equal size, sequences in order.
// Every workgroup works it out from the lengths, so nothing is planned on the
// host and a replayed graph follows them.
struct Chunk {
  int b, i, n;    // sequence (-1: none), its chunk, its length
  int cnt, size;  // the sequence's chunks, the keys of one
  int c0;         // the sequence's first chunk
};
LOOM_DEV int chunk_keys(const StepParams& p, int64_t total) {
  const int64_t per = (total + p.chunks - 1) / p.chunks;
  return (int)min((int64_t)1 << 30, max((int64_t)2, (per + kKeys - 1) / kKeys) * kKeys);
}
// The next larger t.  It ends: the first t gives at most p.chunks + B chunks, p.most
// is at least 2 B where it is set, so t grows by less than half (random batches took
// up to nine tries, most one).
LOOM_DEV int more_keys(int t) { return t + max(kKeys, t / 32 / kKeys * kKeys); }
LOOM_DEV int wave_scan(int v, int lane) {   // inclusive
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(v, m);
    if (lane >= m) v += o;
  }
  return v;
}
LOOM_DEV int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
LOOM_DEV Chunk find_chunk(const StepParams& p, int c) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Chunk r{-1, 0, 0, 1, 0, 0};
  if (p.B <= 64) {          // each wave by itself: one load, no barrier
    const int n = lane < p.B ? seq_len(p, lane) : 0;
    int t = chunk_keys(p, wave_sum64(n)), cnt, inc;
    for (;; t = more_keys(t)) {
      cnt = (n + t - 1) / t;
      inc = wave_scan(cnt, lane);
      if (__builtin_amdgcn_readlane(inc, 63) <= p.most) break;
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(c < inc);
    if (m == 0) return r;
    r.b = __builtin_ctzll(m);
    r.n = __builtin_amdgcn_readlane(n, r.b);
    r.cnt = __builtin_amdgcn_readlane(cnt, r.b);
    r.c0 = __builtin_amdgcn_readlane(inc, r.b) - r.cnt;
  } else {
    __shared__ int64_t s_sum[kThreads / 64];
    __shared__ int s_cnt[kThreads / 64], s_r[4];
    int64_t total = 0;
    for (int b = tid; b < p.B; b += kThreads) total += seq_len(p, b);
    total = wave_sum64(total);
    if (lane == 0) s_sum[wave] = total;
    if (tid == 0) s_r[0] = -1;
    __syncthreads();
    int t = chunk_keys(p, s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3]);
    int base = 0;
    for (int b0 = 0; b0 < p.B; b0 += kThreads) {
      const int b = b0 + tid;
      const int n = b < p.B ? seq_len(p, b) : 0;
      int cnt, inc, all;
      for (;; t = more_keys(t)) {   // (p.most is set up to 256 sequences only)
        cnt = (n + t - 1) / t;
        inc = wave_scan(cnt, lane);
        if (lane == 63) s_cnt[wave] = inc;
        __syncthreads();
        all = s_cnt[0] + s_cnt[1] + s_cnt[2] + s_cnt[3];
        if (all <= p.most) break;
        __syncthreads();
      }
      int at = base + inc - cnt;
      for (int x = 0; x < wave; ++x) at += s_cnt[x];
      if (c >= at && c < at + cnt) {
        s_r[0] = b;
        s_r[1] = n;
        s_r[2] = cnt;
        s_r[3] = at;
      }
      base += all;
      __syncthreads();
      if (c < base) break;
    }
    r.b = __builtin_amdgcn_readfirstlane(s_r[0]);
    if (r.b < 0) return r;
    r.n = __builtin_amdgcn_readfirstlane(s_r[1]);
    r.cnt = __builtin_amdgcn_readfirstlane(s_r[2]);
    r.c0 = __builtin_amdgcn_readfirstlane(s_r[3]);
  }
  r.i = c - r.c0;
  // no more than t (a multiple of 64 that gives cnt of them), so none is empty
  r.size = ((r.n + r.cnt - 1) / r.cnt + kKeys - 1) / kKeys * kKeys;
  return r;
}

// ids received round-robin by the eight XCDs -> contiguous ranges for each
LOOM_DEV int xcd_range(int id, int n) {
  const int x = id & 7, q = n >> 3, r = n & 7;
  return x * q + min(x, r) + (id >> 3);
}

template <int D, bool F16, bool WT>
__global__ void __launch_bounds__(kThreads, D > 128 ? 1 : 2) cache_split_kernel(StepParams p) {
  __shared__ __attribute__((aligned(1024))) char smem[2 * 4 * kKeys * D];
  Part a;
  int tile;                 // rows of the tile this part runs on
  const int id = blockIdx.x;
  if (id < p.nprefix) {     // a prefix part: row tiles of the same keys side by side
    const int x = xcd_range(id, p.nprefix);
    const int rt = x % p.ntp, s = x / p.ntp % p.nsp, g = x / (p.ntp * p.nsp);
    const int rows = p.B * p.H;
    tile = p.rtp;
    a.k = p.pk + (int64_t)g * p.D * p.P;
    a.v = p.pv + (int64_t)g * p.P * p.D;
    a.ld = p.P;
    a.s0 = s * p.tile_p;
    a.s1 = min(p.P, a.s0 + p.tile_p);
    a.i0 = rt * tile;
    a.rows = min(tile, rows - a.i0);
    a.g = g;
    a.once = false;
    a.out0 = ((int64_t)s * p.G + g) * rows + a.i0;
    a.score = nullptr;
  } else {                  // a chunk of a sequence's own keys
    const int x = id - p.nprefix, per = p.G * p.nht;
    const Chunk c = find_chunk(p, x / per);
    if (c.b < 0) return;
    const int g = x % per / p.nht, ht = x % p.nht;
    const int64_t bg = (int64_t)c.b * p.G + g;
    if (c.i == 0 && x % per == 0 && threadIdx.x == 0) p.plan[c.b] = int2{c.c0, c.cnt};
    tile = p.H <= 32 ? 32 : p.H <= 64 ? 64 : 128;
    a.k = p.k + bg * p.D * p.S;
    a.v = p.v + bg * p.S * p.D;
    a.ld = p.S;
    a.s0 = c.i * c.size;
    a.s1 = min(c.n, a.s0 + c.size);
    a.g = -1;
    a.once = p.once != 0;
    a.rows = min(128, p.H - ht * 128);
    a.i0 = (int)(bg * p.H) + ht * 128;
    a.out0 = (int64_t)p.nsp * p.B * p.G * p.H + ((int64_t)(x / per) * p.G + g) * p.H + ht * 128;
    a.score = WT ? p.score + (bg * p.H + ht * 128) * p.Sp : nullptr;
  }
  const bool kreg = a.ld % 8 != 0;
  if (tile == 32) {
    if (kreg) run_part<D, F16, WT, 1, 2, true>(p, a, smem);
    else run_part<D, F16, WT, 1, 2, false>(p, a, smem);
  } else if (tile == 64) {
    if (kreg) run_part<D, F16, WT, 1, 1, true>(p, a, smem);
    else run_part<D, F16, WT, 1, 1, false>(p, a, smem);
  } else {
    if (kreg) run_part<D, F16, WT, 2, 1, true>(p, a, smem);
    else run_part<D, F16, WT, 2, 1, false>(p, a, smem);
  }
}

// ---------------------------------------------------------------------------
// The parts of a row joined, and the weights
// ---------------------------------------------------------------------------
struct Splits {             // a row's partial rows: the prefix's, then its own
  int64_t R, pre0, own0;    // pre0 + s R: prefix part s; own0 + s G H: its own part s
  int nsp, n, GH;
};
LOOM_DEV Splits row_splits(const StepParams& p, int b, int g, int h) {
  Splits s;
  s.R = (int64_t)p.B * p.G * p.H;
  s.pre0 = ((int64_t)g * p.B + b) * p.H + h;
  // (both loaded at once: of a sequence without keys the plan is not written)
  const int len = seq_len(p, b);
  const int2 pl = p.plan[b];
  s.nsp = p.nsp;
  s.GH = p.G * p.H;
  s.own0 = s.nsp * s.R + ((int64_t)pl.x * p.G + g) * p.H + h;
  s.n = s.nsp + (len > 0 ? pl.y : 0);
  return s;
}
LOOM_DEV int64_t split_at(const Splits& s, int u) {
  return u < s.nsp ? u * s.R + s.pre0 : s.own0 + (int64_t)(u - s.nsp) * s.GH;
}

constexpr int kJoinMax = 64;

// CH parts of a thread, u0, u0 + NG, ...: every load at once, then (max, sum, row)
template <int CH>
LOOM_DEV void join_parts(const StepParams& p, const Splits& sp, int u0, int NG, int d, float& M,
                         float& den, f32x4_t& acc) {
  f32x4_t l[CH], o[CH];
#pragma unroll
  for (int u = 0; u < CH; ++u) {
    const int64_t at = split_at(sp, min(u0 + u * NG, sp.n - 1));   // clamped: weight 0
    l[u] = p.ml[at];
    o[u] = *reinterpret_cast<const f32x4_t*>(p.o + at * p.D + d);
  }
  float mc = M;
#pragma unroll
  for (int u = 0; u < CH; ++u) {
    // a part without a key of finite score takes no part (its l is 0, not NaN)
    if (u0 + u * NG >= sp.n || l[u][2] == 0.f) l[u][0] = -INFINITY;
    mc = fmaxf(mc, l[u][0]);
  }
  const float base = mc == -INFINITY ? 0.f : mc;
  const float r = fast_exp2(M - base);
  den *= r;
  acc *= r;
  M = mc;
#pragma unroll
  for (int u = 0; u < CH; ++u) {
    const float w = fast_exp2(l[u][0] - base);
    den += w != 0.f ? w * l[u][2] : 0.f;
    acc += w != 0.f ? o[u] * w : f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
}

// out of a row's (max, sum, row); a row without a finite score is zero
template <bool F16>
LOOM_DEV void store_row(const StepParams& p, int64_t row, int d, float den, const f32x4_t& acc) {
  const float inv = den != 0.f ? 1.f / den : 0.f;
  *reinterpret_cast<u32x2_t*>(p.out + row * p.D + d) =
      u32x2_t{pack2<F16>(acc[0] * inv, acc[1] * inv), pack2<F16>(acc[2] * inv, acc[3] * inv)};
}

// Many rows: D / 4 threads to a row, each over all of its parts.
template <bool F16>
LOOM_DEV void join_rows(const StepParams& p, int x) {
  const int TPR = p.D / 4, RPW = kThreads / TPR;
  const int sub = (int)threadIdx.x / TPR, row = x * RPW + sub;
  if (sub >= RPW || row >= p.B * p.G * p.H) return;
  const int d = ((int)threadIdx.x - sub * TPR) * 4;
  const int bg = row / p.H, h = row - bg * p.H, b = p.G == 1 ? bg : bg / p.G, g = bg - b * p.G;
  const Splits sp = row_splits(p, b, g, h);
  float M = -INFINITY, den = 0.f;
  f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int u0 = 0; u0 < sp.n; u0 += 4) join_parts<4>(p, sp, u0, 1, d, M, den, acc);
  store_row<F16>(p, row, d, den, acc);
}

// Few rows: one workgroup per row, its threads in groups of D / 4 (four d each),
// group y taking parts y, y + NG, ...; the groups' (max, sum, row) meet in LDS.
template <bool F16>
LOOM_DEV void join_row(const StepParams& p, int row) {
  __shared__ f32x4_t s_acc[256];
  __shared__ float s_m[kJoinMax], s_den[kJoinMax];
  const int D = p.D;
  const int bg = row / p.H, h = row - bg * p.H, b = p.G == 1 ? bg : bg / p.G, g = bg - b * p.G;
  const Splits sp = row_splits(p, b, g, h);
  const int ns = sp.n;
  const int TPR = D / 4, NG = min(256 / TPR, kJoinMax);
  const int grp = (int)threadIdx.x / TPR, d = ((int)threadIdx.x - grp * TPR) * 4;
  float M = -INFINITY, den = 0.f;
  f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (grp < NG && grp < ns) {
    if (ns <= NG) {
      join_parts<1>(p, sp, grp, NG, d, M, den, acc);
    } else if (ns <= 2 * NG) {
      join_parts<2>(p, sp, grp, NG, d, M, den, acc);
    } else if (ns <= 4 * NG) {
      join_parts<4>(p, sp, grp, NG, d, M, den, acc);
    } else {
      for (int u0 = grp; u0 < ns; u0 += 8 * NG) join_parts<8>(p, sp, u0, NG, d, M, den, acc);
    }
    s_acc[threadIdx.x] = acc;
    if (d == 0) {
      s_m[grp] = M;
      s_den[grp] = den;
    }
  }
  __syncthreads();
  if (grp != 0) return;
  const int ng = min(NG, ns);
  float Mt = -INFINITY;
  for (int y = 0; y < ng; ++y) Mt = fmaxf(Mt, s_m[y]);
  const float base = Mt == -INFINITY ? 0.f : Mt;
  float dt = 0.f;
  f32x4_t at = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int y = 0; y < ng; ++y) {
    const float w = fast_exp2(s_m[y] - base);
    dt += s_den[y] * w;
    at += s_acc[y * TPR + (int)threadIdx.x] * w;
  }
  store_row<F16>(p, row, d, dt, at);
}

// The keys j0 .. j0 + p.wkeys - 1 of one (b, g): weights_out = weights + sum over
// its heads of 2^(score - M) / l, M and l the row's base and sum over all its parts.
// A lane takes four keys, the workgroup's 1024 / wkeys groups of lanes every so many
// heads; a group's first scores are on their way while M and l are found, two to
// eight threads to a head.  They wait for the length: loads behind it, of scores
// that no key has, cost more (B32 H32 of 4096 to 8192 keys 41.2 -> 39.8 us).
LOOM_DEV void add_weights(const StepParams& p, int bg, int j0) {
  constexpr int HB = 256, HN = 8, UN = 8;
  __shared__ float s_M[HB], s_inv[HB];
  __shared__ f32x4_t s_w[kThreads];
  const int wkeys = p.wkeys, NG = 1024 / wkeys, LPG = wkeys / 4;
  const int tid = threadIdx.x, grp = tid / LPG, lg = tid - grp * LPG;
  const int j = min(j0 + 4 * lg, p.Sp - 4);    // Sp is a multiple of 64: whole pieces
  const float* const score = p.score + (int64_t)bg * p.H * p.Sp + j;
  f32x4_t sc[HN];
  auto load = [&](int h0, int hn) {            // heads h0 + grp + NG x below hn
#pragma unroll
    for (int x = 0; x < HN; ++x)
      if (h0 + NG * x < hn)                    // (the same for all groups)
        sc[x] = *reinterpret_cast<const f32x4_t*>(
            score + (int64_t)min(h0 + grp + NG * x, hn - 1) * p.Sp);
  };
  const int b = p.G == 1 ? bg : bg / p.G, g = bg - b * p.G;
  const int len = seq_len(p, b);
  if (j0 >= len) return;
  load(0, min(p.H, HB));
  const Splits sp0 = row_splits(p, b, g, 0);
  float w_in[4];                               // of keys j0 + tid, 256 apart
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (256 * u < wkeys) w_in[u] = p.w[(int64_t)bg * p.S + min(j0 + 256 * u + tid, len - 1)];
  f32x4_t sum = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // threads to a head: as many as leave 256 threads a head each
  const int tph = p.H <= 32 ? 8 : p.H <= 64 ? 4 : 2, hpp = kThreads / tph;
  for (int hb = 0; hb < p.H; hb += HB) {
    const int hn = min(p.H, hb + HB);
    if (hb > 0) load(hb, hn);
#pragma unroll 1
    for (int h0 = hb; h0 < hn; h0 += hpp) {
      const int h = h0 + tid / tph, y = tid & (tph - 1);
      float M = -INFINITY, L = 0.f;
      if (h < hn) {
        Splits sp = sp0;
        sp.pre0 += h;
        sp.own0 += h;
#pragma unroll 1
        for (int u0 = y; u0 < sp.n; u0 += UN * tph) {
          f32x2_t l[UN];
#pragma unroll
          for (int x = 0; x < UN; ++x)
            l[x] = *reinterpret_cast<const f32x2_t*>(
                p.ml + split_at(sp, min(u0 + x * tph, sp.n - 1)));
          float m = M;
#pragma unroll
          for (int x = 0; x < UN; ++x) {
            // a part without a key of finite score takes no part (its sum is 0)
            if (u0 + x * tph >= sp.n || l[x][1] == 0.f) l[x] = f32x2_t{-INFINITY, 0.f};
            m = fmaxf(m, l[x][0]);
          }
          const float base = m == -INFINITY ? 0.f : m;
          L *= fast_exp2(M - base);
#pragma unroll
          for (int x = 0; x < UN; ++x) L += l[x][1] * fast_exp2(l[x][0] - base);
          M = m;
        }
      }
      for (int x = 1; x < tph; x <<= 1) {
        const float M2 = __shfl_xor(M, x), L2 = __shfl_xor(L, x);
        const float m = fmaxf(M, M2), base = m == -INFINITY ? 0.f : m;
        L = L * fast_exp2(M - base) + L2 * fast_exp2(M2 - base);
        M = m;
      }
      if (y == 0 && h < hn) {
        s_M[h - hb] = M == -INFINITY ? 0.f : M;
        s_inv[h - hb] = L != 0.f ? 1.f / L : 0.f;
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int h0 = hb; h0 < hn; h0 += NG * HN) {
      if (h0 > hb) load(h0, hn);
#pragma unroll
      for (int x = 0; x < HN; ++x) {
        const int h = h0 + grp + NG * x;
        if (h < hn) {
          const float M = s_M[h - hb], inv = s_inv[h - hb];
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] += fast_exp2(sc[x][i] - M) * inv;
        }
      }
    }
    __syncthreads();
  }
  s_w[tid] = sum;
  __syncthreads();
  const float* const f = reinterpret_cast<const float*>(s_w);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int e = 256 * u + tid;
    if (e < wkeys && j0 + e < len) {
      float w = 0.f;
      for (int x = 0; x < NG; ++x) w += f[x * wkeys + e];
      p.w_out[(int64_t)bg * p.S + j0 + e] = w_in[u] + w;
    }
  }
}

// p.njoin workgroups of rows and, with weights, those of every (b, g)'s keys; what
// takes longest first: rows where a thread walks all parts of one (flat), else
// the weights (B32 S8192 39.7 us a step against 42.8 the other way round, B16
// H71 19.6 against 21.0).
template <bool F16, bool WT>
__global__ void __launch_bounds__(256) cache_join_kernel(StepParams p) {
  int x = blockIdx.x;
  if constexpr (WT) {
    const int nw = (p.S + p.wkeys - 1) / p.wkeys, all = p.B * p.G * nw;
    const int y = p.flat ? x - p.njoin : x;    // the weights' workgroup
    if (y >= 0 && y < all) {
      const int bg = y / nw;
      add_weights(p, bg, (y - bg * nw) * p.wkeys);
      return;
    }
    if (!p.flat) x -= all;
  }
  if (p.flat) join_rows<F16>(p, x);
  else join_row<F16>(p, x);
}

// The launch's shape, from the extents alone.
struct Shape {
  int nht, chunks, most, rtp, ntp, nsp, tile_p, nprefix;
  int64_t max_chunks, Sp, rows;
};

Shape shape_of(int64_t B, int64_t G, int64_t H, int64_t D, int64_t P, int64_t S) {
  Shape s{};
  // Workgroups that a launch is sized for: what runs at once, one a CU past D 128 and
  // two up to it.  Up to D 64 three would fit (164 registers, 32 KB), but sizes for
  // 768 gain without a prefix (B32 H32 of 4096 to 8192 keys 22.1 -> 19.4 us a step, B32
  // G8 H8 of 1024 to 4096 41.8 -> 38.9) and lose under one or with equal lengths (B16 G8
  // H4 P4095 S2048 18.6 -> 20.6, B57 H32 of 8000 keys 31.7 -> 33.2)
  const int64_t slots = D > 128 ? 256 : 512;
  s.nht = H <= 32 ? 1 : (int)cdiv64(H, 128);
  s.Sp = cdiv64(S, kKeys) * kKeys;
  if (P > 0) {
    const int64_t rows = B * H;
    // 128 rows share a stage once there are eight stages of them for every CU
    // (G8 B48 H8 P16384: 50 us of split kernel against 68 with 64); below, twice
    // as many tiles over half as many splits, whose sums cost more than the
    // stages (B32 H32 P8192 21.8 us against 25.0, P2048 14.4 against 15.8)
    s.rtp = rows <= 32 ? 32 : G * cdiv64(rows, 128) * cdiv64(P, kKeys) < 8 * 256 ? 64 : 128;
    s.ntp = (int)cdiv64(rows, s.rtp);
    // splits for half of the workgroups, the own keys' parts run beside them (D256
    // B32 G8 H4 P4096 S2048: all of them 98.5 us a step, half 86.2), and at most 64,
    // whose parts a row joins in one round of loads: with up to 256 B1 H32 takes
    // 19.3 us at P16384 against 16.6 and 28.3 at 65536 against 25.0, though 36.2 at
    // 131072 against 47.1 (G2 H16 P65536 29.3 against 31.3)
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(slots / 2 / (G * s.ntp), 64));
    s.tile_p = (int)(cdiv64(std::max<int64_t>(cdiv64(P, want), 2 * kKeys), kKeys) * kKeys);
    s.nsp = (int)cdiv64(P, s.tile_p);
    s.nprefix = (int)(G * s.ntp * s.nsp);
  }
  // Chunks of the whole batch: one round of workgroups, less about what rounding up
  // to whole chunks adds to it (B32 of 4096 to 8192 keys with weights: 46.1 us at
  // 512 chunks, of which 16 wait for a second round, against 39.9).  Rounding up
  // adds anything up to B - 1, so without a prefix, whose parts run beside them, the
  // chunks grow until they are no more than a round (B57 H32 of 8000 keys 513
  // workgroups 64.6 us, 456 of them 52.7; B47 G4 H2 D80 of 3056 keys 564 54.3, 376
  // 44.0; B11 G8 H5 D256 of 4032 keys 264 of 256 99.0, 176 75.8).  With few chunks to
  // a sequence two rounds, which even out their sizes better (B48 G8 of 1024 to 4096
  // keys 116 against 107 us), unless prefix parts fill the gaps
  const int64_t each = std::max<int64_t>(1, slots / (G * s.nht));
  s.chunks = (int)(each >= 2 * B ? each - B * 5 / 8 : P > 0 ? each : 2 * each);
  s.most = each >= 2 * B && P == 0 ? (int)each : INT_MAX;
  s.max_chunks = s.chunks + B;
  s.rows = s.nsp * B * G * H + s.max_chunks * G * H;
  return s;
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
  if (S > (1 << 29) || P > (1 << 29) || !loom_prod_le({B, G}, 65535) ||
      !loom_prod_le({B, G, H}, 1 << 23) || !loom_prod_le({B, G, S, D}, (int64_t)1 << 50) ||
      !loom_prod_le({G, P, D}, (int64_t)1 << 50) ||
      (weights && !loom_prod_le({B, G, cdiv64(S, 128)}, 1 << 23)))
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
  const size_t need = loom_hip_cache_decode_workspace_bytes(B, G, H, D, P, S, weights != nullptr);
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_decode: workspace needs %zu bytes (16-byte aligned), got %zu", need,
                     workspace_bytes);
  // The workspace is written while tensors are read, out and weights_out while
  // lens, weights and the workspace are: a shared byte gives results that depend on
  // the order of workgroups.  Two are safe: weights_out on weights (every element is
  // read and written by one thread) and out on q (read before the join writes)
  const int64_t cache = B * G * S * D * 2, prefix = G * P * D * 2, rows = B * G * H * D * 2,
                summed = B * G * S * 4;
  const LoomSpan in[] = {{prefix_k, prefix}, {prefix_v, prefix}, {k, cache}, {v, cache},
                         {lens, B * 4}, {out == q ? nullptr : q, rows},
                         {weights_out == weights ? nullptr : weights, summed}},
                 outs[] = {{out, rows}, {weights_out, summed}, {workspace, (int64_t)need}};
  if (loom_outputs_overlap(in, outs))
    return loom_fail(err, errlen, LOOM_EINVAL,
                     "cache_decode: out, weights_out and the workspace must not overlap the other "
                     "tensors or each other (but weights_out may be weights, out may be q)");
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
  const Shape s = shape_of(B, G, H, D, P, S);
  char* ws = static_cast<char*>(workspace);
  p.plan = reinterpret_cast<int2*>(ws);
  ws += align256((size_t)B * 8);
  p.ml = reinterpret_cast<f32x4_t*>(ws);
  ws += align256((size_t)s.rows * 16);
  p.o = reinterpret_cast<float*>(ws);
  ws += align256((size_t)s.rows * D * 4);
  p.score = reinterpret_cast<float*>(ws);
  p.B = (int)B;
  p.G = (int)G;
  p.H = (int)H;
  p.D = (int)D;
  p.P = (int)P;
  p.S = (int)S;
  p.Sp = (int)s.Sp;
  p.nht = s.nht;
  p.chunks = s.chunks;
  p.most = s.most;
  p.rtp = s.rtp;
  p.ntp = s.ntp;
  p.nsp = s.nsp;
  p.tile_p = s.tile_p;
  p.nprefix = s.nprefix;
  // Several rows to a workgroup where rows are many or their parts few: B60 G8 H16
  // P1584 39.0 -> 28.1 us a step, B30 G8 H12 P976 with weights 25.0 -> 21.0; but
  // 1024 rows of 32 parts 24.5 -> 29.7
  const int64_t parts = s.nsp + cdiv64(s.chunks, B);
  p.flat = B * G * H > 2048 || (B * G * H >= 1024 && parts <= 16);
  p.njoin = (int)(p.flat ? cdiv64(B * G * H, kThreads / (D / 4)) : B * G * H);
  p.once = s.nht == 1 && 4 * B * G * S * D > (int64_t)256 << 20;
  // Keys of a workgroup that gathers weights: many spread the heads' statistics over
  // more of them and leave fewer groups without a head (G256 in all, H4 S4096 118,
  // 105, 98 and 95 us a step with 128, 256, 512 and 1024, H32 146, 135, 133 and 131;
  // B32 H32 S8192 42.0, 40.0, 38.8 and 39.9), as long as they leave workgroups for
  // the CUs (B1 S4096 12.9 against 13.3 with 128 and 256, B16 H32 S4096 18.1 against
  // 19.8 with 256 and 512)
  auto parts_of = [&](int64_t keys) { return B * G * cdiv64(S, keys); };
  p.wkeys = parts_of(1024) >= 1024 ? 1024 : parts_of(512) >= 256 ? 512 : parts_of(256) >= 256 ? 256 : 128;
  p.c2 = scale * 1.4426950408889634f;
  if (loom_validate_only()) return loom_ok(err, errlen);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(s.nprefix + s.max_chunks * G * s.nht)), block(kThreads);
  // the kernel built for 64, 128 or 256 (the next one up) runs any narrower D
  auto split = [&](auto kern) { hipLaunchKernelGGL(kern, grid, block, 0, st, p); };
  if (weights) {
    if (D > 128) split(cache_split_kernel<256, F16, true>);
    else if (D > 64) split(cache_split_kernel<128, F16, true>);
    else split(cache_split_kernel<64, F16, true>);
  } else {
    if (D > 128) split(cache_split_kernel<256, F16, false>);
    else if (D > 64) split(cache_split_kernel<128, F16, false>);
    else split(cache_split_kernel<64, F16, false>);
  }
  int rc = loom_check_launch(err, errlen, "cache_decode (split)");
  if (rc) return rc;
  if (weights)
    hipLaunchKernelGGL((cache_join_kernel<F16, true>),
                       dim3((unsigned)(p.njoin + B * G * cdiv64(S, p.wkeys))), block, 0, st, p);
  else
    hipLaunchKernelGGL((cache_join_kernel<F16, false>), dim3((unsigned)p.njoin), block, 0, st, p);
  return loom_check_launch(err, errlen, "cache_decode (join)");
}

}  // namespace

extern "C" {

size_t loom_hip_cache_decode_workspace_bytes(int64_t B, int64_t G, int64_t H, int64_t D, int64_t P,
                                             int64_t S, int weights) {
  if (B <= 0 || G <= 0 || H <= 0 || D <= 0 || P < 0 || S <= 0) return 0;
  // what does not fit is reported as no size at all fits
  if (P > (1 << 29) || S > (1 << 29) || D > (1 << 20) || !loom_prod_le({B, G}, 65535) ||
      !loom_prod_le({B, G, H}, 1 << 23))
    return SIZE_MAX;
  const Shape s = shape_of(B, G, H, D, P, S);
  return align256((size_t)B * 8) + align256((size_t)s.rows * 16) +
         align256((size_t)s.rows * D * 4) + (weights ? (size_t)(B * G * H * s.Sp) * 4 : 0);
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
