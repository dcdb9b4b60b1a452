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
//
// gfx950 mapping.  The rows of a (b, g) are its tokens' heads, t-major, cut into tiles of
// 32 to 256: H heads share a token's keys, so a tile of 256 rows of 4 heads spans 64
// tokens and reads window + 64 keys, not window + 256.  A tile walks the blocks of 64
// keys that any of its rows sees: the sinks', those at the edges of the window (masked),
// then those that all rows see, by code of its own without the masks' branches.  Taken
// together they cost those blocks the overlap of products and exponentials (when it was
// built, a window of 4096 over 8192 tokens of 64 heads 1290 us against 1087, and prompts of
// 4096 tokens of 128 heads under 1024 + 4 keys 379 against 332: a sixth of the blocks are
// edges.  Now 1040 to 1110 us, 1.0 PFLOP/s as attention.hip without a window, and 309 to
// 335).  Few rows over many keys (a step) share a tile's blocks between workgroups, which a
// second launch joins; a step is bound by streaming the window (B32 G8 H4 f16 window 4096:
// 490 MB in 82 us, 6.0 TB/s; of D 256, whose tiles of 32 rows take every vector register, 980
// MB in 158 us).
// Rounding: scores, bases and sums are fp32 (scale log2 e multiplies the fp32 score: q
// times it, rounded, would cost a steep row two digits); p is rounded to 16 bits for its
// product with v, and out divided by the sum of the rounded p.  f16, which loses bits
// below 2^-14, holds p 2^7 times larger.
#include "common.h"

#include <cmath>
#include <type_traits>

namespace {

constexpr int kKeys = 64;         // keys per stage

struct WindowParams {
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  const int* lens;
  const int* counts;
  uint16_t* out;
  f32x2_t* ml;      // per partial row (split, b g, row): base, sum of p
  float* o;         // per partial row: sum of p v, D values
  int B, G, H, D, T, S;
  int window, sinks;
  int ntiles, nsplit;
  int once;         // the caches are read by non-temporal copies
  int koff32;       // D * S * 2 < 2^32: K's per-lane DMA offsets fit 32 bits
  float c2;         // scale * log2(e)
};

// What a tile of rows reads: sequence b's rows (t, h), t-major, r0 .. r0 + rows - 1
// of c H, and the blocks of 64 keys that any of them sees: nsb blocks of sinks, then
// those from wb0 on.
struct Tile {
  int r0, rows;
  int p0;           // position of token 0
  int low, ns;      // seen keys: j < ns, and low <= j <= pmax
  int pmin, pmax;
  int nsb, wb0, nblk;
  int mb0, mb1;     // blocks mb0 .. mb1 - 1: keys that all rows see
  int nedge;        // blocks ahead of these in the order that they are taken in
};
LOOM_DEV Tile tile_of(const WindowParams& p, int b, int tile, int RT) {
  Tile a;
  // (the same for the workgroup, stated to the compiler: addresses follow from them)
  const int n = __builtin_amdgcn_readfirstlane(min(max(p.lens[b], 0), p.S));
  const int c =
      __builtin_amdgcn_readfirstlane(p.counts ? min(max(p.counts[b], 0), p.T) : p.T);
  a.r0 = tile * RT;
  a.rows = min(RT, c * p.H - a.r0);
  a.p0 = n - c;
  a.pmin = a.p0 + a.r0 / p.H;
  a.pmax = a.p0 + (a.r0 + a.rows - 1) / p.H;
  a.low = max(0, a.pmin - p.window + 1);
  a.ns = min(min(p.sinks, a.low), a.pmax + 1);
  a.nsb = (max(a.ns, 0) + kKeys - 1) / kKeys;
  a.wb0 = max(a.low / kKeys, a.nsb);
  const int end = a.pmax < 0 ? a.wb0 : max(a.wb0, a.pmax / kKeys + 1);
  a.nblk = a.pmax < 0 ? 0 : a.nsb + end - a.wb0;
  a.mb0 = max(a.wb0, (max(0, a.pmax - p.window + 1) + kKeys - 1) / kKeys);
  a.mb1 = max(0, a.pmin + 1) / kKeys;
  if (a.mb1 <= a.mb0) a.mb0 = a.mb1 = end;
  a.nedge = a.nblk - (a.mb1 - a.mb0);
  return a;
}
// The block that is taken i-th: the sinks', those at the window's edges, then those that
// all rows see.
LOOM_DEV int tile_block(const Tile& a, int i) {
  if (i >= a.nedge) return a.mb0 + i - a.nedge;
  if (i < a.nsb) return i;
  const int kb = a.wb0 + i - a.nsb;
  return kb < a.mb0 ? kb : kb + (a.mb1 - a.mb0);
}

// W / KG waves of 16 QT rows each share 64-key stages of K and V copied by LDS DMA
// (K through registers where its rows start off 16-byte boundaries, KREG), NS of
// them.  KG 2: two waves share 16 QT rows, each taking one 32-key half of every
// stage, and merge at the end.  The MFMAs compute
//   S^T[key, row] = K^T . Q^T,   O^T[d, row] += V^T . P^T,
// both row operands by transposed LDS reads; softmax in fp32 in the log2 domain
// with a lazily moved base.  WPE: waves per SIMD the registers must allow; DC: the
// head dim that is computed, for narrower heads in the stages of D.  SPLIT: the
// tile's blocks are shared by p.nsplit workgroups, whose sums window_join_kernel
// joins.
template <int D, int QT, int W, bool F16, bool KREG, bool SPLIT, int KG, int NS, int WPE, int DC>
__global__ void __launch_bounds__(64 * W, WPE) window_tile_kernel(WindowParams p) {
  static_assert(KG == 1 || KG == 2, "a stage has two 32-key halves");
  constexpr int RT = 16 * QT * W / KG;          // rows per workgroup
  constexpr int K_BYTES = D * kKeys * 2, V_BYTES = kKeys * D * 2;
  constexpr int K_INSTR = K_BYTES / 1024 / W, V_INSTR = V_BYTES / 1024 / W;
  static_assert(K_INSTR >= 1 && V_INSTR >= 1, "every wave issues K and V copies");
  constexpr int LPW = (KREG ? 0 : K_INSTR) + V_INSTR;
  constexpr int VROW = D * 2, V_ROWS_PER_I = 1024 / VROW;
  constexpr int DSTEPS = DC / 32, DT = DC / 16;
  static_assert(LPW * (NS - 2) <= 63, "vmcnt range");
  constexpr bool QDMA = D <= 128;
  constexpr int QROW = D * 2;
  constexpr int Q_LDS = QDMA ? RT * QROW : 0;
  constexpr int Q_INSTR = QDMA ? Q_LDS / 1024 / W : 0;
  static_assert(!QDMA || Q_LDS % (1024 * W) == 0, "whole Q copies per wave");
  constexpr int STAGE = K_BYTES + V_BYTES;
  static_assert(NS * STAGE + Q_LDS <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) char smem[NS * STAGE + Q_LDS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qw = wave / KG, kh = wave % KG;     // rows and key half of this wave
  const int r = lane & 15, g = lane >> 4;
  const int a4 = r >> 2, c4 = r & 3;            // transposed-read lane roles

  // ids go round-robin to the eight XCDs: each takes whole (b, g)s, whose tiles follow
  // each other and share their keys in its L2
  const int BG = p.B * p.G;
  int bg, tile, split = 0;
  {
    const int per = p.ntiles * (SPLIT ? p.nsplit : 1);
    int x;
    if (BG % 8 == 0) {
      const int j = blockIdx.x >> 3;
      bg = j / per * 8 + (blockIdx.x & 7);
      x = j % per;
    } else {
      const int id = xcd_remap(blockIdx.x, BG * per);
      bg = id / per;
      x = id - bg * per;
    }
    tile = x;
    if constexpr (SPLIT) {
      tile = x / p.nsplit;
      split = x - tile * p.nsplit;
    }
  }
  const int b = bg / p.G, gh = bg - b * p.G, H = p.H;
  const Tile a = tile_of(p, b, tile, RT);
  if (a.rows <= 0) return;
  const int Dr = p.D, S = p.S;
  const int i0 = SPLIT ? (int)((int64_t)a.nblk * split / p.nsplit) : 0;
  const int i1 = SPLIT ? (int)((int64_t)a.nblk * (split + 1) / p.nsplit) : a.nblk;
  const int nblk = i1 - i0;
  const uint16_t* __restrict__ kg = p.k + (int64_t)bg * Dr * S;
  const uint16_t* __restrict__ vg = p.v + (int64_t)bg * S * Dr;
  // row lr of the tile in q's and out's [B T G H] rows
  auto row_of = [&](int lr) {
    const int x = a.r0 + lr, t = x / H;
    return (((int64_t)b * p.T + t) * p.G + gh) * H + (x - t * H);
  };
  auto first_key = [&](int blk) { return tile_block(a, i0 + blk) * kKeys; };

  auto stK = [&](int s) { return (lds_char_t*)(smem + s * STAGE); };
  auto stV = [&](int s) { return (lds_char_t*)(smem + s * STAGE + K_BYTES); };
  lds_char_t* const sQ = (lds_char_t*)(smem + NS * STAGE);
  // ---- DMA of block `blk` into stage s.  Ks rows d >= Dr come from zeros; V chunks
  // past Dr repeat the row's last.  A block that holds keys that no row sees clamps
  // K's pieces to the row (those keys are masked) and takes the V rows of such keys
  // from zeros: they may hold anything, and a weight of zero times NaN is NaN.
  uint32_t koff[K_INSTR], voff[V_INSTR];
#pragma unroll
  for (int i = 0; i < K_INSTR; ++i) {
    const int j = wave * K_INSTR + i, d = j * 8 + lane / 8;
    // unsigned: it wraps (and goes unused, koff32 == 0) when D * S * 2 >= 2^32
    koff[i] = ((uint32_t)d * (uint32_t)S + (uint32_t)(((lane % 8) ^ k_swz(d)) * 8)) * 2u;
  }
#pragma unroll
  for (int i = 0; i < V_INSTR; ++i) {
    const int j = wave * V_INSTR + i, kr = j * V_ROWS_PER_I + lane / (D / 8);
    voff[i] = (uint32_t)(kr * Dr + min((lane % (D / 8)) ^ v_swz<D>(kr), Dr / 8 - 1) * 8) * 2;
  }
  // (tiles of few rows only: keys of larger ones are shared)
  const bool once = KG == 2 && p.once != 0;
  auto issue = [&](int s, int blk) __attribute__((always_inline)) {
    const int kv0 = first_key(blk);
    const uint32_t lk = lds_addr(stK(s)), lv = lds_addr(stV(s));
    const bool whole = kv0 + kKeys - 1 <= a.pmax && (kv0 >= a.low || kv0 + kKeys <= a.ns);
    if (whole && !once && (KREG || p.koff32)) {           // wave-uniform
      if constexpr (!KREG) {
#pragma unroll
        for (int i = 0; i < K_INSTR; ++i) {
          const int j = wave * K_INSTR + i;
          if (j * 8 < Dr)
            dma_load16_s(koff[i], kg + kv0, __builtin_amdgcn_readfirstlane(lk + j * 1024));
          else
            dma_load16(loom_zero_kb + lane * 4, __builtin_amdgcn_readfirstlane(lk + j * 1024));
        }
      }
#pragma unroll
      for (int i = 0; i < V_INSTR; ++i)
        dma_load16_s(voff[i], vg + (int64_t)kv0 * Dr, __builtin_amdgcn_readfirstlane(lv + (wave * V_INSTR + i) * 1024));
      return;
    }
    const int ln = KG == 2 ? lane : fresh(lane);
    if constexpr (!KREG) {
#pragma unroll
      for (int i = 0; i < K_INSTR; ++i) {
        const int j = wave * K_INSTR + i;
        const int d = j * 8 + ln / 8;
        const int key = min(kv0 + ((ln % 8) ^ k_swz(d)) * 8, S - 8);
        const uint16_t* from = kg + (int64_t)d * S + key;
        if (j * 8 >= Dr) dma_load16(loom_zero_kb + ln * 4, __builtin_amdgcn_readfirstlane(lk + j * 1024));
        else if (once) dma_once16(from, __builtin_amdgcn_readfirstlane(lk + j * 1024));
        else dma_load16(from, __builtin_amdgcn_readfirstlane(lk + j * 1024));
      }
    }
#pragma unroll
    for (int i = 0; i < V_INSTR; ++i) {
      const int j = wave * V_INSTR + i;
      const int kr = j * V_ROWS_PER_I + ln / (D / 8);
      const int key = kv0 + kr;
      const bool seen = key <= a.pmax && (key >= a.low || key < a.ns);
      const void* from = seen ? (const void*)((const char*)(vg + (int64_t)kv0 * Dr) + voff[i])
                              : (const void*)(loom_zero_kb + ln * 4);
      if (once) dma_once16(from, __builtin_amdgcn_readfirstlane(lv + j * 1024));
      else dma_load16(from, __builtin_amdgcn_readfirstlane(lv + j * 1024));
    }
  };
  // ---- KREG: K pieces of block `blk` into registers, then into stage s
  const rsrc_t krs = make_rsrc(kg, KREG ? (uint32_t)(Dr * S * 2) : 0u);
  u32x4_t kr[KREG ? K_INSTR : 1];
  auto kload = [&](int blk) __attribute__((always_inline)) {
    const int kv0 = first_key(blk);
#pragma unroll
    for (int i = 0; i < K_INSTR; ++i) {
      const int j = wave * K_INSTR + i;
      const int d = j * 8 + lane / 8;
      kr[i] = j * 8 < Dr ? row_piece8(krs, S, d, kv0 + ((lane % 8) ^ k_swz(d)) * 8)
                         : u32x4_t{0u, 0u, 0u, 0u};
    }
  };
  auto kstore = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < K_INSTR; ++i)
      *reinterpret_cast<__attribute__((address_space(3))) u32x4_t*>(
          stK(s) + (wave * K_INSTR + i) * 1024 + lane * 16) = kr[i];
  };

  // ---- Q by LDS DMA up to D 128 (rows past the tile's repeat its last; chunks past
  // Dr are zeroed when read), ahead of the first stages, then these
  if constexpr (QDMA) {
    const uint32_t lq = lds_addr(sQ);
#pragma unroll
    for (int i = 0; i < Q_INSTR; ++i) {
      const int j = wave * Q_INSTR + i;
      const int e = j * 1024 + lane * 16;
      const int lr = e / QROW, cp = (e % QROW) / 16;
      const int c = min(cp ^ q_swz<D>(lr), Dr / 8 - 1);
      dma_load16(p.q + row_of(min(lr, a.rows - 1)) * Dr + c * 8, lq + j * 1024);
    }
  }
#pragma unroll
  for (int s = 0; s < NS - 1; ++s)
    if (s < nblk) {
      if constexpr (KREG) {
        kload(s);
        kstore(s);
      }
      issue(s, s);
    }
  const int rw0 = 16 * QT * qw;                 // this wave's first row
  u32x4_t qf[DSTEPS][QT];
  if constexpr (!QDMA) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const uint16_t* from = p.q + row_of(min(rw0 + 16 * qt + r, a.rows - 1)) * Dr;
#pragma unroll
      for (int ds = 0; ds < DSTEPS; ++ds) {
        const int d0 = ds * 32 + g * 8;
        const u32x4_t raw = *reinterpret_cast<const u32x4_t*>(from + min(d0, Dr - 8));
        qf[ds][qt] = d0 < Dr ? raw : u32x4_t{0u, 0u, 0u, 0u};
      }
    }
  }
  // the positions of this lane's rows, and of the wave's first and last
  const bool active = rw0 < a.rows;
  int pos[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) pos[qt] = a.p0 + (a.r0 + min(rw0 + 16 * qt + r, a.rows - 1)) / H;
  const int pw0 = __builtin_amdgcn_readfirstlane(a.p0 + (a.r0 + min(rw0, a.rows - 1)) / H);
  const int pw1 = __builtin_amdgcn_readfirstlane(
      a.p0 + (a.r0 + min(rw0 + 16 * QT, a.rows) - 1) / H);

  const float c2 = p.c2;
  float m_run[QT];
  f32x4_t ot[DT][QT], lacc[QT];
  const u32x4_t ones = u32x4_t{kOnePair<F16>, kOnePair<F16>, kOnePair<F16>, kOnePair<F16>};
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m_run[qt] = 0.f;
    lacc[qt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) ot[dt][qt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  bool first = true;        // some row's base is not set yet
  // log2 of what the largest p starts at, and how far it may rise: f16 loses bits
  // below 2^-14 (bf16 has fp32's exponents)
  constexpr float kLift = F16 ? 7.f : 0.f, kRise = kLift + 8.f;

  // Whether rows of the wave see other keys of a half than other rows of the tile do.
  // (Rows of one token see the same; and what no row sees lies there as zeros.)
  auto mixed_half = [&](int k0) __attribute__((always_inline)) {
    return a.pmin != a.pmax &&
           (k0 + 31 > pw0 || (k0 <= pw1 - p.window && k0 + 31 >= a.low));
  };
  constexpr uint32_t kInf = F16 ? 0x7c00 : 0x7f80;
  bool odd = false;         // such a half held an infinity or NaN

  // The wave's rows against a stage's keys; EDGE: some of them are not seen by some rows.
  // (Without the edges' branches the other blocks' products and exponentials overlap.)
  auto compute = [&](int s, int kv0, auto any) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(any)::value;
    const lds_char_t* ks = stK(s);
    const lds_char_t* vs = stV(s);
#pragma unroll
    for (int hh = 0; hh < 2 / KG; ++hh) {
      const int h = KG == 1 ? hh : kh;
      const int k0 = kv0 + 32 * h;              // this half's keys: k0 .. k0 + 31
      // a half that no row of the wave sees
      if (EDGE && (k0 > pw1 || (k0 + 31 <= pw0 - p.window && k0 >= p.sinks))) continue;
      // ---- S^T = K^T Q^T; st[j][qt][i] = score of key k0 + 16 j + 4 g + i
      f32x4_t st[2][QT];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) st[j][qt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ds = 0; ds < DSTEPS; ++ds) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int jt = 2 * h + j;
          const int d = ds * 32 + g * 8 + a4;               // & 3 == a4
          const int ch = (2 * jt + (c4 >> 1)) ^ k_swz(d);
          const lds_char_t* q = ks + d * (kKeys * 2) + ch * 16 + (c4 & 1) * 8;
          const u32x2_t lo = lds_read_tr16(q);
          const u32x2_t hi = lds_read_tr16(q + 4 * (kKeys * 2));
          const u32x4_t kf = u32x4_t{lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) st[j][qt] = mfma16t<F16>(kf, qf[ds][qt], st[j][qt]);
        }
      }
      // ---- log2-domain scores relative to the base; keys that a row does not see
      // are -inf
      float lmax[QT];
      bool big = false;
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st[j][qt][i] = __builtin_fmaf(st[j][qt][i], c2, -m_run[qt]);
        if constexpr (EDGE) {
          // (no short circuits: a branch for every key takes longer than a comparison)
          const int ps = fresh(pos[qt]), lo = max(0, ps - p.window + 1);
          const int at0 = k0 + 4 * g - lo, n = max(0, ps + 1 - lo), sk = min(p.sinks, ps + 1) - lo;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int at = at0 + 16 * j + i;
              const bool sees = ((uint32_t)at < (uint32_t)n) | (at < sk);
              st[j][qt][i] = sees ? st[j][qt][i] : -INFINITY;
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, st[j][qt][i]);
        lmax[qt] = mx;
        big |= mx > kRise;
      }
      // ---- lazy online softmax: a row's base is set by its first half with a finite
      // score and moves (O and the sum rescale) when a score rises 2^8 above it
      if (first || __builtin_amdgcn_ballot_w64(big) != 0) {
        bool left = false;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          float mx = lmax[qt];
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const bool unset = first && lacc[qt][0] == 0.f;
          const float shift = unset ? (mx == -INFINITY ? 0.f : mx - kLift) : fmaxf(mx - kLift, 0.f);
          const float alpha = unset ? 1.f : fast_exp2(-shift);
          lacc[qt] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) ot[dt][qt] *= alpha;
          m_run[qt] += shift;
#pragma unroll
          for (int j = 0; j < 2; ++j) st[j][qt] -= shift;
          left |= unset && mx == -INFINITY;
        }
        first = __builtin_amdgcn_ballot_w64(left) != 0;
      }
      // ---- O^T += V^T P^T and l += ones . P^T over these 32 keys
      u32x4_t pf[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        f32x4_t e0, e1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e0[i] = fast_exp2(st[0][qt][i]);
          e1[i] = fast_exp2(st[1][qt][i]);
        }
        pf[qt] = u32x4_t{pack2<F16>(e0[0], e0[1]), pack2<F16>(e0[2], e0[3]),
                         pack2<F16>(e1[0], e1[1]), pack2<F16>(e1[2], e1[3])};
        lacc[qt] = mfma16t<F16>(ones, pf[qt], lacc[qt]);
      }
      auto v_op = [&](int dt) {
        const int k0r = 32 * h + 4 * g + a4;
        const int ch = (2 * dt + (c4 >> 1)) ^ v_swz<D>(k0r);
        const lds_char_t* q = vs + k0r * VROW + ch * 16 + (c4 & 1) * 8;
        const u32x2_t lo = lds_read_tr16(q);                // keys k0 + 4 g + 0..3
        const u32x2_t hi = lds_read_tr16(q + 16 * VROW);    // keys k0 + 16 + 4 g + 0..3
        return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
      };
      // Keys that some rows of the tile see and the wave's do not all: a weight of zero
      // times an infinity or NaN of theirs would reach rows that do not see them.  Such
      // values are looked for (the largest magnitude's bits, two elements at a time);
      // where there are any they count as zeros here, and the rows that see them get them
      // behind the loop.
      if (EDGE && mixed_half(k0)) {
        typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
        u16x2_t top = u16x2_t{0, 0};
#pragma unroll
        for (int i = 0; i < 32 * VROW / 1024; ++i) {
          const u32x4_t w = *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(
              vs + 32 * h * VROW + i * 1024 + fresh(lane) * 16);
#pragma unroll
          for (int x = 0; x < 4; ++x)
            top = __builtin_elementwise_max(top,
                                            __builtin_bit_cast(u16x2_t, w[x] & 0x7fff7fffu));
        }
        if (__builtin_amdgcn_ballot_w64(top[0] >= kInf || top[1] >= kInf) != 0) {
          odd = true;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            u32x4_t vf = v_op(dt);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              // (an exponent of all ones carries into the sign's place)
              const uint32_t bad =
                  ((vf[x] & kInf * 0x10001u) + (F16 ? 0x04000400u : 0x00800080u)) & 0x80008000u;
              vf[x] &= ~((bad >> 15) * 0xffffu);
            }
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) ot[dt][qt] = mfma16t<F16>(vf, pf[qt], ot[dt][qt]);
          }
          continue;
        }
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u32x4_t vf = v_op(dt);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) ot[dt][qt] = mfma16t<F16>(vf, pf[qt], ot[dt][qt]);
      }
    }
  };

  // ---- pipeline: NS stages (the first NS-1 issued above), waits placed by hand.  (Not
  // unrolled over the stages: their addresses would not leave registers enough.)
  auto landed = [&](int it) __attribute__((always_inline)) {
    if (min(NS - 2, nblk - 1 - it) >= 1) LOOM_WAIT_VMCNT(LPW);
    else LOOM_WAIT_VMCNT(0);
    // this wave's reads of the stage that is overwritten next, and KREG's stores
    LOOM_WAIT_LGKM0();
    barrier_nofence();
  };
  if constexpr (QDMA) {
    if (nblk > 0) {
      landed(0);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const int lr = rw0 + 16 * qt + r;
#pragma unroll
        for (int ds = 0; ds < DSTEPS; ++ds) {
          const u32x4_t raw = *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(
              sQ + lr * QROW + ((4 * ds + g) ^ q_swz<D>(lr)) * 16);
          qf[ds][qt] = ds * 32 + g * 8 < Dr ? raw : u32x4_t{0u, 0u, 0u, 0u};
        }
      }
    }
  }
  int s = 0;
  auto step = [&](int it, auto any) __attribute__((always_inline)) {
    landed(it);
    const int to = s == 0 ? NS - 1 : s - 1;     // the stage of block it - 1
    const bool ahead = it + NS - 1 < nblk;
    if constexpr (KREG) {
      if (ahead) kload(it + NS - 1);
    }
    if (ahead) issue(to, it + NS - 1);
    if (active) compute(s, first_key(it), any);
    if constexpr (KREG) {
      if (ahead) kstore(to);
    }
    s = s == NS - 1 ? 0 : s + 1;
  };
  // the edges, then, by code without their branches, the rest
  const int nedge = min(max(a.nedge - i0, 0), nblk);
#pragma unroll 1
  for (int it = 0; it < nedge; ++it) step(it, std::true_type{});
#pragma unroll 1
  for (int it = nedge; it < nblk; ++it) step(it, std::false_type{});

  // (without a block nothing has waited for the Q copies)
  if (nblk == 0) LOOM_WAIT_VMCNT(0);
  // ---- infinities and NaN that counted as zeros, to the rows that see them
  if (odd) {
#pragma unroll 1
    for (int it = 0; it < nblk; ++it) {
#pragma unroll 1
      for (int x = 0; x < kKeys; ++x) {
        const int key = first_key(it) + x, k0 = key & ~31;
        if ((KG == 2 && (x >> 5) != kh) || !mixed_half(k0) || key > a.pmax ||
            (key < a.low && key >= a.ns))
          continue;
        const uint16_t* from = vg + (int64_t)key * Dr;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w = from[min(16 * dt + 4 * g + i, Dr - 1)];
            if ((w & kInf) != kInf) continue;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
              if ((key <= pos[qt]) & ((key > pos[qt] - p.window) | (key < p.sinks)))
                ot[dt][qt][i] += lo16<F16>(w);
          }
      }
    }
  }
  // ---- a row without a key of finite score is zero, whatever its keys' v held
  bool none = false;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) none |= lacc[qt][0] == 0.f;
  if (__builtin_amdgcn_ballot_w64(none) != 0) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
      if (lacc[qt][0] == 0.f)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) ot[dt][qt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // ---- KG 2: the pair's second wave hands its state over through the idle stages
  // (lane by lane: both hold the same rows and columns); a half that saw no key (l =
  // 0) takes no part
  if constexpr (KG == 2) {
    constexpr int SLOT = QT * (DT + 1) * 64;    // f32x4 per wave: O, then (l, m)
    static_assert(W / 2 * SLOT * 16 <= NS * STAGE, "merge area");
    LOOM_WAIT_VMCNT(0);
    LOOM_WAIT_LGKM0();
    barrier_nofence();
    f32x4_t* const mg = reinterpret_cast<f32x4_t*>(smem) + qw * SLOT + lane;
    if (kh == 1) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) mg[(qt * (DT + 1) + dt) * 64] = ot[dt][qt];
        mg[(qt * (DT + 1) + DT) * 64] = f32x4_t{lacc[qt][0], m_run[qt], 0.f, 0.f};
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
      m_run[qt] = M;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        ot[dt][qt] = ot[dt][qt] * f0 + mg[(qt * (DT + 1) + dt) * 64] * f1;
    }
  }

  // ---- ot[dt][qt][i] is d = 16 dt + 4 g + i of row rw0 + 16 qt + r
  if constexpr (SPLIT) {
    const int64_t base = ((int64_t)split * BG + bg) * ((int64_t)p.T * H) + a.r0;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int lr = rw0 + 16 * qt + r;
      if (lr < a.rows) {
        if (g == 0) p.ml[base + lr] = f32x2_t{m_run[qt], lacc[qt][0]};
        float* to = p.o + (base + lr) * Dr;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          if (dt * 16 + 4 * g < Dr) *reinterpret_cast<f32x4_t*>(to + dt * 16 + 4 * g) = ot[dt][qt];
      }
    }
    return;
  }
  // out = O / l (a row without a key of finite score is zero).  With D <= 128 and rows
  // of exactly D, each wave stages its rows in its own slice of the Q region and writes
  // them back as whole rows, 16 bytes a lane.
  if constexpr (QDMA && DC == D) {
    if (Dr == D) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const float inv = lacc[qt][0] != 0.f ? 1.f / lacc[qt][0] : 0.f;
        const int lr = rw0 + 16 * qt + r;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const f32x4_t o = ot[dt][qt];
          const int at = (2 * dt + (g >> 1)) ^ q_swz<D>(lr);
          *reinterpret_cast<__attribute__((address_space(3))) u32x2_t*>(
              sQ + lr * QROW + at * 16 + (g & 1) * 8) =
              u32x2_t{pack2<F16>(o[0] * inv, o[1] * inv), pack2<F16>(o[2] * inv, o[3] * inv)};
        }
      }
      constexpr int CPR = QROW / 16;
      lds_order();
#pragma unroll
      for (int k = 0; k < 16 * QT * CPR / 64; ++k) {
        const int idx = k * 64 + lane;
        const int lr = rw0 + idx / CPR, cp = idx % CPR;
        const u32x4_t v = *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(
            sQ + lr * QROW + cp * 16);
        if (lr < a.rows)
          *reinterpret_cast<u32x4_t*>(p.out + row_of(lr) * Dr + (cp ^ q_swz<D>(lr)) * 8) = v;
      }
      return;
    }
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float inv = lacc[qt][0] != 0.f ? 1.f / lacc[qt][0] : 0.f;
    const int lr = rw0 + 16 * qt + r;
    if (lr < a.rows) {
      uint16_t* to = p.out + row_of(lr) * Dr;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const f32x4_t o = ot[dt][qt];
        if (dt * 16 + 4 * g < Dr)
          *reinterpret_cast<u32x2_t*>(to + dt * 16 + 4 * g) =
              u32x2_t{pack2<F16>(o[0] * inv, o[1] * inv), pack2<F16>(o[2] * inv, o[3] * inv)};
      }
    }
  }
}

// The partial sums of a row joined: D / 4 threads to a row, four d each.
template <bool F16>
__global__ void __launch_bounds__(256) window_join_kernel(WindowParams p) {
  const int TPR = p.D / 4, RPW = 256 / TPR;
  const int sub = (int)threadIdx.x / TPR;
  const int64_t R = (int64_t)p.T * p.H, all = R * p.B * p.G;
  const int64_t row = (int64_t)blockIdx.x * RPW + sub;      // (b g, t, h)
  if (sub >= RPW || row >= all) return;
  const int bg = (int)(row / R), x = (int)(row - bg * R), t = x / p.H, h = x - t * p.H;
  const int b = bg / p.G, g = bg - b * p.G;
  const int c = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  if (t >= c) return;
  const int d = ((int)threadIdx.x - sub * TPR) * 4;
  float M = -INFINITY, den = 0.f;
  f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int CH = 4;
  for (int s0 = 0; s0 < p.nsplit; s0 += CH) {
    f32x2_t ml[CH];
    f32x4_t o[CH];
#pragma unroll
    for (int s = 0; s < CH; ++s) {
      const int64_t at = min(s0 + s, p.nsplit - 1) * all + row;
      ml[s] = p.ml[at];
      o[s] = *reinterpret_cast<const f32x4_t*>(p.o + at * p.D + d);
    }
    float m = M;
#pragma unroll
    for (int s = 0; s < CH; ++s) {
      // a part without a key of finite score takes no part (its sum is 0, not NaN)
      if (s0 + s >= p.nsplit || ml[s][1] == 0.f) ml[s][0] = -INFINITY;
      m = fmaxf(m, ml[s][0]);
    }
    const float base = m == -INFINITY ? 0.f : m;
    const float r = fast_exp2(M - base);
    den *= r;
    acc *= r;
    M = m;
#pragma unroll
    for (int s = 0; s < CH; ++s) {
      const float w = fast_exp2(ml[s][0] - base);
      den += w != 0.f ? w * ml[s][1] : 0.f;
      acc += w != 0.f ? o[s] * w : f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
  const int64_t to = (((int64_t)b * p.T + t) * p.G + g) * p.H + h;
  *reinterpret_cast<u32x2_t*>(p.out + to * p.D + d) =
      u32x2_t{pack2<F16>(acc[0] * inv, acc[1] * inv), pack2<F16>(acc[2] * inv, acc[3] * inv)};
}

// The launch's shape, from the extents alone.  (launch_window has the kernels that it gives.)
struct Shape {
  int tile;         // rows of a tile: 32, 64, 128 or 256
  int64_t ntiles;   // per (b, g)
  int nsplit;       // workgroups that share a tile's keys
};
Shape shape_of(int64_t B, int64_t G, int64_t H, int64_t D, int64_t T, int64_t S, int64_t window,
               int64_t sinks) {
  Shape s{};
  const int64_t rows = T * H, BG = B * G;
  // The largest tile that leaves a workgroup to every CU (B4 G8 H4 T4096 window 1024: 256
  // rows 310 us, 128 426; f16 B3 G2 H5 D80 T1001: 64 rows 19.9, 32 27.5, and 128, with 237
  // workgroups, 18.1).  Past
  // D 128 two waves of 16 rows each would not hold a pair's 64 rows without spills.
  const int64_t most = D > 128 ? 128 : 256;
  s.tile = 32;
  while (s.tile < most && s.tile < rows && BG * cdiv64(rows, s.tile * 2) >= 256) s.tile *= 2;
  if (D > 128 && s.tile == 64) s.tile = 32;
  s.ntiles = cdiv64(rows, s.tile);
  // the blocks of keys that a tile reads at most
  const int64_t span = std::min(S, std::min(window, S) + cdiv64(s.tile, H));
  const int64_t blocks = cdiv64(span, kKeys) + 1 + cdiv64(std::min(sinks, S), kKeys);
  // Splits of at least two blocks, as many as run at once (B1 H32 window 512: 5 splits and
  // their join 10.4 us a call, one workgroup 11.0)
  const int64_t slots = D > 128 ? 256 : 512;
  const int64_t want = std::min<int64_t>(slots / (BG * s.ntiles), blocks / 2);
  s.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>(want, 64));
  // Tiles past 32 rows are 256 at least, a round of workgroups.  Exactly 256 are cut in two
  // where two of their workgroups fit a CU, by LDS and registers, and a tile's blocks are
  // worth the join (tiles of 64 rows, G8 H4 T512: D 64 window 2048 24.5 us whole, 29.9 cut,
  // 4096 41.4 and 42.9, 8192 72.7 and 65.1; D 96 29.7 and 37.3, 50.2 and 52.3, 89.2 and 79.7;
  // 256 rows of D 128, T2048 window 1024: 42.9 and 66.3).
  const bool two = s.tile <= (D > 96 ? 32 : D > 64 ? 64 : 128);
  if (s.tile > 32 && !(two && blocks >= 72)) s.nsplit = 1;
  return s;
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

template <bool F16, bool KREG, bool SPLIT>
void launch_window(const WindowParams& p, const Shape& s, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.B * p.G * s.ntiles * s.nsplit)), b4(256), b8(512);
  auto launch = [&](auto kern, dim3 block) { hipLaunchKernelGGL(kern, grid, block, 0, st, p); };
  // a tile that is never split
  auto whole = [&](auto kern, dim3 block) {
    if constexpr (!SPLIT) launch(kern, block);
  };
  // the kernel built for 64, 128 or 256 (the next one up) runs any narrower head
  if (p.D > 128) {
    switch (s.tile) {
      case 32: launch(window_tile_kernel<256, 1, 4, F16, KREG, SPLIT, 2, 2, 1, 256>, b4); break;
      default: whole(window_tile_kernel<256, 1, 8, F16, KREG, false, 1, 2, 1, 256>, b8); break;
    }
  } else if (p.D > 96) {
    switch (s.tile) {
      case 32: launch(window_tile_kernel<128, 1, 4, F16, KREG, SPLIT, 2, 2, 2, 128>, b4); break;
      case 64: whole(window_tile_kernel<128, 1, 8, F16, KREG, false, 2, 2, 2, 128>, b8); break;
      case 128: whole(window_tile_kernel<128, 1, 8, F16, KREG, false, 1, 3, 1, 128>, b8); break;
      default: whole(window_tile_kernel<128, 2, 8, F16, KREG, false, 1, 3, 1, 128>, b8); break;
    }
  } else if (p.D > 64) {
    switch (s.tile) {
      case 32: launch(window_tile_kernel<128, 1, 4, F16, KREG, SPLIT, 2, 2, 2, 96>, b4); break;
      case 64: launch(window_tile_kernel<128, 1, 8, F16, KREG, SPLIT, 2, 2, 2, 96>, b8); break;
      case 128: whole(window_tile_kernel<128, 1, 8, F16, KREG, false, 1, 3, 1, 96>, b8); break;
      default: whole(window_tile_kernel<128, 2, 8, F16, KREG, false, 1, 3, 1, 96>, b8); break;
    }
  } else {
    switch (s.tile) {
      case 32: launch(window_tile_kernel<64, 1, 4, F16, KREG, SPLIT, 2, 2, 2, 64>, b4); break;
      case 64: launch(window_tile_kernel<64, 1, 8, F16, KREG, SPLIT, 2, 2, 2, 64>, b8); break;
      case 128: launch(window_tile_kernel<64, 1, 8, F16, KREG, SPLIT, 1, 3, 1, 64>, b8); break;
      default: whole(window_tile_kernel<64, 2, 8, F16, KREG, false, 1, 3, 1, 64>, b8); break;
    }
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
  const Shape s = shape_of(B, G, H, D, T, S, window, sinks);
  p.ntiles = (int)s.ntiles;
  p.nsplit = s.nsplit;
  // keys that one workgroup reads once, and more of them than the 256 MB last-level
  // cache holds, displace nothing that is read again
  p.once = s.ntiles == 1 &&
           4 * B * G * D * std::min(S, p.window + T + (int64_t)p.sinks) > (int64_t)256 << 20;
  p.koff32 = loom_prod_le({D, S, 2}, 0xffffffffll) ? 1 : 0;
  p.ml = static_cast<f32x2_t*>(workspace);
  p.o = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                 align256((size_t)(s.nsplit * B * G * H * T) * 8));
  if (loom_validate_only()) return loom_ok(err, errlen);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (s.nsplit == 1) {
    if (S % 8) launch_window<F16, true, false>(p, s, st);
    else launch_window<F16, false, false>(p, s, st);
    return loom_check_launch(err, errlen, "window_attention");
  }
  if (S % 8) launch_window<F16, true, true>(p, s, st);
  else launch_window<F16, false, true>(p, s, st);
  int rc = loom_check_launch(err, errlen, "window_attention (split)");
  if (rc) return rc;
  hipLaunchKernelGGL((window_join_kernel<F16>),
                     dim3((unsigned)cdiv64(B * G * H * T, 256 / (D / 4))), dim3(256), 0, st, p);
  return loom_check_launch(err, errlen, "window_attention (join)");
}

}  // namespace

extern "C" {

size_t loom_hip_window_attention_workspace_bytes(int64_t B, int64_t G, int64_t H, int64_t D,
                                                 int64_t T, int64_t S, int64_t window,
                                                 int64_t sinks) {
  if (B <= 0 || G <= 0 || H <= 0 || D <= 0 || T <= 0 || S <= 0 || window <= 0 || sinks < 0) return 0;
  // what does not fit is reported as no size at all fits
  if (S > (1 << 29) || D > (1 << 20) || !loom_prod_le({B, G}, 65535) ||
      !loom_prod_le({T, H}, 1 << 29) || !loom_prod_le({B, G, cdiv64(T * H, 32)}, 1 << 23))
    return SIZE_MAX;
  const Shape s = shape_of(B, G, H, D, T, S, window, sinks);
  if (s.nsplit == 1) return 0;
  const size_t rows = (size_t)(s.nsplit * B * G * H * T);
  return align256(rows * 8) + align256(rows * D * 4);
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
