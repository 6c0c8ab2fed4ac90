// Streams of weights for a few token rows (device code of decode.hip and
// fp4_mm.hip).
//
// A few rows stream every weight they meet once and do almost nothing with it, so
// these kernels are weight rows through v_mfma_f32_16x16x32_bf16: A = 16 weight rows x
// 32 columns, B = up to 16 token rows.  Both come by LDS DMA, each wave issuing its
// own stages' (stream_items), or the token rows' once for the workgroup (lock_items).
// What bounds them is requests in flight: 80 to 110 KB per CU here reach 5.4 to 6
// TB/s.  Loads into registers instead (16 rows x 64 bytes an instruction, two units
// of 128 columns per wave) reached 4.9 TB/s on rows of 4 KB and 2.7 on 1.5 KB: half
// lines, and a unit's registers in flight only.
#pragma once

#include "common.h"
#include "dma_asm.h"
#include "fp4.h"
#include "gemm_common.h"
#include "probe.h"

namespace ttamd {
namespace decode {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kLds = 160 * 1024;

// W_FP4_8: 4-bit tiles by their upper or lower 8 rows, two tiles of a row of tiles at a
// time (for a workgroup that owns 8 output rows).
enum WeightType { W_BF16 = 0, W_FP4 = 1, W_FP4_8 = 2 };
constexpr int load_rows(int wt) { return wt == W_FP4 ? 16 : 8; }

// Weights [E, N, K]: bf16 rows, or 4-bit tiles and their exponents (fp4.hip).
struct Weights {
  const void* w;
  const uint8_t* exps;
};

// ---- streams: every wave pulls its own weight rows through a ring in LDS --------
// A stage of a wave: its weight rows and the token rows over kCols columns (bf16: a
// 128-byte line of every row; 4 bits: one tile, or two halves, and the exponents).  A
// DMA instruction moves 8 bf16 weight rows, one 4-bit tile of 16, or 8 (4, 2) token
// rows of 128 (256, 512) bytes; BL and NB count the instructions.
template <int WT, int BL, int NB, int NS>
struct Ring {
  static constexpr int kCols = WT == W_BF16 ? 64 : WT == W_FP4 ? 128 : 256;
  static constexpr int kBlocks = WT == W_BF16 ? (BL + 1) / 2 : BL;  // of 16 rows
  static constexpr int kExps = BL * 1024;                           // 4 bits: 256 bytes of exponents per block
  static constexpr int kRowsAt = kExps + (WT == W_BF16 ? 0 : 256 * BL);
  static constexpr int kBytes = kRowsAt + 1024 * NB;
  static constexpr int kOps = (WT == W_BF16 ? BL : 2 * BL) + NB;
  static constexpr int kRows = NB * (512 / kCols);
  static constexpr int NT = (kRows + 15) / 16;
  static constexpr int kAll = kWaves * NS * kBytes;
  static_assert(WT != W_FP4_8 || BL == 1);
};

// One item of a wave: rows of one expert (or the shared one) times its token rows.
template <int BL>
struct Item {
  uint64_t base[BL];  // per load: bf16, its first row of 8; 4 bits, its first tile
  uint64_t exps[BL];  // 4 bits: its exponents
  uint64_t x;         // where the offsets of its token rows start
  int lo, cnt;        // token rows lo .. cnt - 1
  int start;          // their first place in the caller's order; -1: the shared expert
  int rb;             // which run of rows (the caller's)
  int K;
  int pair;           // lock_items' last round: which pair of the run (the caller's)
  bool live;          // the wave has rows here
};

// The DMAs of stage s of BL 4-bit blocks: their tiles, then the exponents of the
// tiles' group of four.
template <int BL>
__device__ __forceinline__ void issue_tiles(const Item<BL>& c, int s, uint32_t at, int exps_at) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int b = 0; b < BL; ++b) dma::dma16((uint32_t)(16 * l), c.base[b] + (uint64_t)s * 1024, at + b * 1024);
#pragma unroll
  for (int b = 0; b < BL; ++b)
    dma::dma4((uint32_t)(4 * l), c.exps[b] + (uint64_t)(s >> 2) * 256, at + exps_at + b * 256);
}

// acc += stage cs of BL 4-bit blocks (tiles and exponents at st) times NT tiles of 16
// of its token rows (256 bytes each at rows_at, chunk c of row r at c ^ r); ROWS: how
// many rows the stage holds.
template <int BL, int NT, int ROWS, int ALL, class Free>
__device__ __forceinline__ void consume_tiles(floatx4_t (&acc)[BL][ALL], const char* st, int exps_at,
                                              const char* rows_at, int cs, int left, Free free) {
  const int l = threadIdx.x & 63, n = l & 15, q = l >> 4;
  uint4 qw[BL];
  float scale[BL];
  bf16x8_t bx[4][NT];
#pragma unroll
  for (int b = 0; b < BL; ++b) {
    qw[b] = *(const uint4*)(st + b * 1024 + 16 * l);
    scale[b] = fp4_scale(*(const uint32_t*)(st + exps_at + b * 256 + 4 * l), cs & 3);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = (16 * t + n) & (ROWS - 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) bx[j][t] = *(const bf16x8_t*)(rows_at + r * 256 + (((4 * q + j) ^ (r & 15)) << 4));
  }
  free();
  if (left < 128 && 32 * q >= left) {  // (codes past the row's end are zeros; so must be what they meet)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int t = 0; t < NT; ++t) bx[j][t] = __builtin_bit_cast(bf16x8_t, make_uint4(0u, 0u, 0u, 0u));
  }
#pragma unroll
  for (int b = 0; b < BL; ++b) {
    const uint32_t d[4] = {qw[b].x, qw[b].y, qw[b].z, qw[b].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8_t aw = fp4_frag(d[j], scale[b]);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        acc[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(aw, bx[j][t], acc[b][t], 0, 0, 0);
    }
  }
}

// acc += stage cs of 8 rows' halves of two tiles times the token rows (512 bytes each).
template <int ROWS, class Free>
__device__ __forceinline__ void consume_halves(floatx4_t& acc, const char* st, int exps_at, const char* rows_at, int cs,
                                               int left, Free free) {
  const int l = threadIdx.x & 63, n = l & 15, q = l >> 4, r = n & (ROWS - 1);
  const uint32_t ex = *(const uint32_t*)(st + exps_at + 4 * l);
  uint4 qw[2];
  bf16x8_t bx[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    qw[h] = *(const uint4*)(st + (32 * h + 8 * q + (n & 7)) * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) bx[h][j] = *(const bf16x8_t*)(rows_at + r * 512 + (((16 * h + 4 * q + j) ^ r) << 4));
  }
  free();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (128 * h >= left) break;
    if (128 * h + 32 * q >= left) {
#pragma unroll
      for (int j = 0; j < 4; ++j) bx[h][j] = __builtin_bit_cast(bf16x8_t, make_uint4(0u, 0u, 0u, 0u));
    }
    const uint32_t d[4] = {qw[h].x, qw[h].y, qw[h].z, qw[h].w};
    const float scale = fp4_scale(ex, (2 * cs + h) & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp4_frag(d[j], scale), bx[h][j], acc, 0, 0, 0);
  }
}

// Runs the items first, first + step, ... < nitems.  Of a item's stages the wave
// takes every KS-th from ks on.  The DMAs run over the flattened sequence of all
// its stages, NS ahead, so neither an epilogue nor the next expert's start empties
// the pipe, and no wave waits for another here.  item_of(i): the i-th item; its
// token rows go kRows at a time: origin(item, n0) is where the bytes of rows from n0
// on are counted from, src(item, n0, i) those of row i; done(item, c0, rows, acc):
// the sums of rows c0 .. c0 + rows - 1 (lane l, block b, tile t: weight rows
// 4 (l / 16) .. + 3, token row c0 + 16 t + l % 16).
template <int WT, int BL, int NB, int NS, class ItemOf, class Origin, class Src, class Done>
__device__ __forceinline__ void stream_items(char* ring, int first, int step, int nitems, int ks, int KS,
                                             ItemOf item_of, Origin origin, Src src, Done done) {
  using namespace dma;
  using R = Ring<WT, BL, NB, NS>;
  constexpr int NT = R::NT, MB = R::kBlocks;
  const int l = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = l & 15, q = l >> 4;
  ring += w * (NS * R::kBytes);
  const uint32_t lds0 = lds_addr(ring);

  // 16-byte chunk of its row that lane l moves in instruction i: LDS holds chunk c
  // of row r at c ^ cswz(r) (8 chunks a row) or c ^ r (16), so that the fragment
  // reads of 16 rows meet no bank twice
  auto chunk8 = [&](int i) { return (l & 7) ^ cswz(8 * i + (l >> 3)); };
  auto chunk16 = [&](int i) { return (l & 15) ^ ((4 * i + (l >> 4)) & 15); };
  auto chunk32 = [&](int i) { return (l & 31) ^ ((2 * i + (l >> 5)) & 15); };
  auto row_of = [&](int i) {
    return WT == W_BF16 ? 8 * i + (l >> 3) : WT == W_FP4 ? 4 * i + (l >> 4) : 2 * i + (l >> 5);
  };
  auto chunk_of = [&](int i) { return WT == W_BF16 ? chunk8(i) : WT == W_FP4 ? chunk16(i) : chunk32(i); };

  // the issuing end
  int it = first, n0 = 0, s = ks;
  bool more = it < nitems;
  Item<BL> in;
  uint32_t va[BL], vb[NB];
  uint64_t xbase = 0;
  auto rows = [&]() __attribute__((always_inline)) {
    xbase = origin(in, n0);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      vb[b] = src(in, n0, min(n0 + row_of(b), in.cnt - 1)) + (uint32_t)(16 * chunk_of(b));
    }
  };
  auto enter = [&]() __attribute__((always_inline)) {  // item `it`, or the next with a stage for this wave
    for (;; it += step) {
      more = it < nitems;
      if (!more) return;
      in = item_of(it);
      if (in.live && in.cnt > in.lo && ks * R::kCols < in.K) break;
    }
    n0 = in.lo, s = ks;
    if constexpr (WT == W_BF16) {
#pragma unroll
      for (int i = 0; i < BL; ++i) va[i] = (uint32_t)((l >> 3) * in.K * 2) + (uint32_t)(16 * chunk8(i));
    }
  };
  auto issue = [&](int slot) __attribute__((always_inline)) {
    const uint32_t at = lds0 + (uint32_t)(slot * R::kBytes);
    const int left = in.K - s * R::kCols;  // columns of the row from this stage on, a multiple of 32
    if constexpr (WT == W_BF16) {
      const uint64_t k = (uint64_t)s * 128;
      if (left >= 64) {
#pragma unroll
        for (int i = 0; i < BL; ++i) dma16(va[i], in.base[i] + k, at + i * 1024);
#pragma unroll
        for (int b = 0; b < NB; ++b) dma16(vb[b], xbase + k, at + R::kRowsAt + b * 1024);
      } else {  // past the row's end: the chunk 64 bytes before once more
#pragma unroll
        for (int i = 0; i < BL; ++i) dma16(va[i] - (chunk8(i) & 4 ? 64u : 0u), in.base[i] + k, at + i * 1024);
#pragma unroll
        for (int b = 0; b < NB; ++b)
          dma16(vb[b] - (chunk8(b) & 4 ? 64u : 0u), xbase + k, at + R::kRowsAt + b * 1024);
      }
    } else {
      if constexpr (WT == W_FP4) {
        issue_tiles<BL>(in, s, at, R::kExps);
      } else {  // (past the last tile: the first once more)
        const int h = left > 128 ? l >> 5 : 0;
        dma16((uint32_t)(1024 * h + 256 * (l >> 3 & 3) + 16 * (l & 7)), in.base[0] + (uint64_t)s * 2048, at);
        dma4((uint32_t)(4 * (l & 0x37)), in.exps[0] + (uint64_t)(s >> 1) * 256, at + R::kExps);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int ch = chunk_of(b);
        const uint32_t back = 8 * ch >= left ? (uint32_t)(16 * (ch & ~3)) : 0u;
        dma16(vb[b] - back, xbase + (uint64_t)s * (2 * R::kCols), at + R::kRowsAt + b * 1024);
      }
    }
    s += KS;
    if (s * R::kCols < in.K) return;
    s = ks;
    n0 += R::kRows;
    if (n0 >= in.cnt) {
      it += step;
      enter();
    }
    if (more) rows();
  };
  enter();
  if (more) rows();
  int ahead = 0;
#pragma unroll 1  // (one copy of the code: a cold instruction cache is what a small call waits for)
  for (; ahead < NS && more; ++ahead) issue(ahead);

  // the consuming end
  int slot = 0;
  for (int ci = first; ci < nitems; ci += step) {
    const Item<BL> c = item_of(ci);
    for (int c0 = c.lo; c0 < c.cnt; c0 += R::kRows) {
      floatx4_t acc[MB][NT];
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[b][t] = floatx4_t{0.f, 0.f, 0.f, 0.f};
      if (c.live)
        for (int cs = ks; cs * R::kCols < c.K; cs += KS) {
          if (ahead == NS) wait_vm<(NS - 1) * R::kOps>();
          else wait_vm<0>();
          const char* st = ring + slot * R::kBytes;
          const int left = c.K - cs * R::kCols;
          if constexpr (WT == W_BF16) {
            bf16x8_t aw[MB][2], bx[2][NT];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int ch = 4 * h + q;
#pragma unroll
              for (int b = 0; b < MB; ++b) {  // (the second half of a last block of 8 rows: the first once more)
                const int r = 16 * b + (2 * b + 1 < BL ? n : n & 7);
                aw[b][h] = *(const bf16x8_t*)(st + r * 128 + ((ch ^ cswz(r)) << 4));
              }
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                const int r = (16 * t + n) & (R::kRows - 1);
                bx[h][t] = *(const bf16x8_t*)(st + R::kRowsAt + r * 128 + ((ch ^ cswz(r)) << 4));
              }
            }
            lds_wait();  // the slot is free
            if (more) issue(slot);
            else --ahead;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h == 1 && left < 64) break;
#pragma unroll
              for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int b = 0; b < MB; ++b)
                  acc[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(aw[b][h], bx[h][t], acc[b][t], 0, 0, 0);
            }
          } else {
            auto free = [&]() __attribute__((always_inline)) {
              lds_wait();
              if (more) issue(slot);
              else --ahead;
            };
            const char* rows_at = st + R::kRowsAt;
            if constexpr (WT == W_FP4) consume_tiles<BL, NT, R::kRows>(acc, st, R::kExps, rows_at, cs, left, free);
            else consume_halves<R::kRows>(acc[0][0], st, R::kExps, rows_at, cs, left, free);
          }
          slot = slot == NS - 1 ? 0 : slot + 1;
        }
      done(c, c0, min(c.cnt - c0, R::kRows), acc);
    }
  }
  wait_vm<0>();
}

// Waves that share an item (log2): rounds of the walk times a wave's stages in one,
// twice; half a stage for a meeting of KS waves, whose 1.5 us of latency pass while the
// next stages load; half an item for the last round, where items of more rows end late.
// From the experts really hit.  (128 experts of 1536 x 2048, 64 tokens, exactly 3 rounds
// of whole pairs: whole 161 us, eighths, which this chooses, 134; 96 rows of 68
// experts in 4 bits: whole 35.0 us, quarters 32.2.)  One round that half the chip's
// waves share already has its requests, and no next stages for a meeting to hide behind
// (41 experts' w13 of 544 x 1440 in 4 bits: whole 12.9 us, quarters 14.4); not so the
// eight waves of a workgroup that walks by itself (5 experts and the shared one, w2 of
// 5120 x 8192: whole 90 us, shared 75).
__host__ __device__ inline int split_log(int items, int slots, int stages, int most) {
  if (slots > kWaves && items <= slots && 2 * items >= slots) return 0;
  int best = 0, cost = 0x7fffffff;
  for (int k = 0; k <= most && (1 << k) <= stages; ++k) {
    const int rounds = ((items << k) + slots - 1) / slots;
    const int st = (stages + (1 << k) - 1) >> k;
    const int c = rounds * (2 * st + (k > 0)) + (rounds > 1 ? st : 0);
    if (c < cost) best = k, cost = c;
  }
  return best;
}

// Load b of an item: load_rows(WT) rows of expert e's [N, K] weights from row `row` on.
template <int WT, int BL>
__device__ __forceinline__ void set_load(Item<BL>& c, int b, const Weights& m, int64_t e, int N, int K, int row) {
  if constexpr (WT == W_BF16) {
    c.base[b] = (uint64_t)((const bf16_t*)m.w + (e * N + row) * K);
  } else {
    const int C = (K + 127) / 128, C4 = (C + 3) / 4;
    const int64_t at = e * ((N + 15) / 16) + row / 16;
    const int half = WT == W_FP4_8 ? row >> 3 & 1 : 0;  // (8 places of 16 and of 4 bytes)
    c.base[b] = (uint64_t)((const char*)m.w + at * C * 1024 + half * 128);
    c.exps[b] = (uint64_t)(m.exps + at * C4 * 256 + half * 32);
  }
}

// The KS partial sums of row pairs (two blocks each), added in order: MR token rows at
// a time (13 rows of 1000 x 1440 in 4 bits: 4 at a time 10.5 us, 16 6.7), two rounds of
// LDS in turn (a round is read before the next one's barrier and written after it).
// emit(item, r, i, quad, v0, v1): rows 4 quad .. + 3 of the blocks of the workgroup's
// pair r, token row i.  Every wave calls it.
constexpr int meet_bytes(int rows) { return 2 * rows * kWaves * 128; }
template <int MR, int BL, int NT, class Emit>
__device__ __forceinline__ void meet_pairs(char* lds, int& turn, int log_ks, const Item<BL>& c, int c0, int rows,
                                           const floatx4_t (&acc)[2][NT], Emit emit) {
  const int tid = threadIdx.x, l = tid & 63, n = l & 15, q = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (log_ks == 0) {
    if (c.live) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (16 * t + n < rows) emit(c, w, c0 + 16 * t + n, q, acc[0][t], acc[1][t]);
    }
    return;
  }
  constexpr int per = 4 * MR;
  for (int m0 = 0; m0 < rows; m0 += MR) {
    floatx4_t* const red = (floatx4_t*)(lds + turn * (meet_bytes(MR) / 2));
    turn ^= 1;
    if (c.live) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int i = 16 * t + n - m0;
        if (i >= 0 && i < MR) {
          red[(w * 2 + 0) * per + i * 4 + q] = acc[0][t];
          red[(w * 2 + 1) * per + i * 4 + q] = acc[1][t];
        }
      }
    }
    dma::lds_barrier();
    // (kWaves per / KS places, at most 256)
    const int r = tid / per, at = tid % per, i = m0 + (at >> 2);
    if (r < kWaves >> log_ks && i < rows) {
      const floatx4_t* v = red + (r << log_ks) * 2 * per + at;
      floatx4_t v0 = v[0], v1 = v[per];
      for (int j = 1; j < 1 << log_ks; ++j) v0 += v[2 * j * per], v1 += v[2 * j * per + per];
      emit(c, r, c0 + i, at & 3, v0, v1);
    }
  }
}

// ---- lock step: 4-bit weights and more token rows -------------------------------
// The token rows of a stage (128 columns, 32 NR rows) are one copy that all waves
// read, each wave holding two tiles of its own, so the workgroup walks the stages
// together, one barrier each; NS - 2 stages stay in flight across it.
template <int NR, int NS>
struct Lock {
  static constexpr int kMine = 2560;  // a wave's two tiles and their exponents
  static constexpr int kRowsAt = kWaves * kMine;
  static constexpr int kBytes = kRowsAt + kWaves * NR * 1024;
  static constexpr int kOps = 4 + NR;
  static constexpr int kRows = 32 * NR;
  static constexpr int NT = 2 * NR;
  static constexpr int kAll = NS * kBytes;
};

// Of n items, those that full rounds of the workgroups take in lock step.  A last
// round that would leave more than a quarter of them idle goes pair by pair instead:
// the eight waves of a workgroup share a pair's stages, and where even the pairs are
// too few, each pair's token rows go in two parts (33 experts' w13 of 4096 x 7168 in 4
// bits, 528 items of 256 workgroups: 187 us in 3 rounds, 119 so).  Four stages per wave
// at least: 33 experts' w2 of 7168 x 2048, two per wave, took 77 us in rounds and 89 so.
__device__ __forceinline__ int lock_rounds(int n, int stages) {
  const int G = gridDim.x, left = n % G;
  return stages >= 4 * kWaves && left > 0 && left <= G * 3 / 4 ? n - left : n;
}
constexpr int kTailNB = 4, kTailNS = 2;  // 16 token rows a pass
using TailRing = Ring<W_FP4, 2, kTailNB, kTailNS>;

// Items and callbacks as stream_items'; item_of(i, r): run i's pair r, for wave r of
// the workgroup (a wave with none takes part with any blocks, its sums dropped).
// emit(item, i, quad, v0, v1): rows 4 quad .. + 3 of the item's pair, token row i.
template <int NR, int NS, class ItemOf, class Origin, class Src, class Emit>
__device__ __forceinline__ void lock_items(char* ring, int all, int stages, ItemOf item_of_pair, Origin origin, Src src,
                                           Emit emit) {
  using namespace dma;
  using L = Lock<NR, NS>;
  constexpr int NT = L::NT;
  const int l = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t lds0 = lds_addr(ring);
  const int nitems = lock_rounds(all, stages), first = blockIdx.x, step = gridDim.x;
  auto item_of = [&](int i) __attribute__((always_inline)) { return item_of_pair(i, w); };
  // the wave's share of the token rows: rows 4 (w + 8 b) + l / 16, chunk c at c ^ row
  auto row_of = [&](int b) { return 4 * (w + kWaves * b) + (l >> 4); };
  auto chunk = [&](int b) { return (l & 15) ^ (row_of(b) & 15); };

  // the issuing end
  int it = first, n0 = 0, s = 0;
  bool more = it < nitems;
  Item<2> in;
  uint32_t vb[NR];
  uint64_t xbase = 0;
  auto rows = [&]() __attribute__((always_inline)) {
    xbase = origin(in, n0);
#pragma unroll
    for (int b = 0; b < NR; ++b)
      vb[b] = src(in, n0, min(n0 + row_of(b), in.cnt - 1)) + (uint32_t)(16 * chunk(b));
  };
  auto enter = [&]() __attribute__((always_inline)) {
    more = it < nitems;
    if (!more) return;
    in = item_of(it);
    n0 = 0, s = 0;
  };
  auto issue = [&](int slot) __attribute__((always_inline)) {
    const uint32_t at = lds0 + (uint32_t)(slot * L::kBytes);
    const int left = in.K - s * 128;
    issue_tiles<2>(in, s, at + w * L::kMine, 2048);
#pragma unroll
    for (int b = 0; b < NR; ++b) {
      const int ch = chunk(b);
      const uint32_t back = 8 * ch >= left ? (uint32_t)(16 * (ch & ~3)) : 0u;
      dma16(vb[b] - back, xbase + (uint64_t)s * 256, at + L::kRowsAt + (w + kWaves * b) * 1024);
    }
    if (++s * 128 < in.K) return;
    s = 0;
    n0 += L::kRows;
    if (n0 >= in.cnt) {
      it += step;
      enter();
    }
    if (more) rows();
  };
  enter();
  if (more) rows();
  int ahead = 0;
#pragma unroll 1
  for (; ahead < NS - 1 && more; ++ahead) issue(ahead);

  // the consuming end
  int slot = 0;
  for (int ci = first; ci < nitems; ci += step) {
    const Item<2> c = item_of(ci);
    for (int c0 = 0; c0 < c.cnt; c0 += L::kRows) {
      const int here = min(c.cnt - c0, L::kRows), tiles = (here + 15) >> 4;
      floatx4_t acc[2][NT];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[b][t] = floatx4_t{0.f, 0.f, 0.f, 0.f};
      for (int cs = 0; cs * 128 < c.K; ++cs) {
        // stage cs has landed, and every wave is done with the one before
        if (ahead == NS - 1) wait_vm_barrier<(NS - 2) * L::kOps>();
        else wait_vm_barrier<0>();
        if (more) issue(slot == 0 ? NS - 1 : slot - 1);  // into the slot of the stage before
        else --ahead;
        const char* st = ring + slot * L::kBytes;
        const int left = c.K - cs * 128;
        const char *mine = st + w * L::kMine, *shared = st + L::kRowsAt;
        auto free = []() __attribute__((always_inline)) {};
        if (tiles <= NT / 2) consume_tiles<2, NT / 2, L::kRows>(acc, mine, 2048, shared, cs, left, free);
        else consume_tiles<2, NT, L::kRows>(acc, mine, 2048, shared, cs, left, free);
        slot = slot == NS - 1 ? 0 : slot + 1;
      }
      if (c.live) {
        const int n = l & 15, q = l >> 4;
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (16 * t + n < here) emit(c, c0 + 16 * t + n, q, acc[0][t], acc[1][t]);
      }
    }
  }
  wait_vm<0>();
  if (nitems == all) return;
  __syncthreads();
  static_assert(TailRing::kAll + meet_bytes(TailRing::kRows) <= L::kAll, "LDS");
  const int pairs = (all - nitems) * kWaves, parts = 2 * pairs <= (int)gridDim.x ? 2 : 1;
  int turn = 0;
  stream_items<W_FP4, 2, kTailNB, kTailNS>(
      ring, blockIdx.x, gridDim.x, pairs * parts, w, kWaves,
      [&](int i) __attribute__((always_inline)) {
        const int pair = i / parts;
        Item<2> c = item_of_pair(nitems + pair / kWaves, pair % kWaves);
        if (parts == 2) {
          const int half = (c.cnt + 1) >> 1;
          if (i & 1) c.lo = half;
          else c.cnt = half;
        }
        return c;
      },
      origin, src,
      [&](const Item<2>& c, int c0, int rows, const floatx4_t (&acc)[2][TailRing::NT]) __attribute__((always_inline)) {
        if (!c.live) return;  // (of the whole workgroup: the item is all waves')
        meet_pairs<TailRing::kRows>(ring + TailRing::kAll, turn, 3, c, c0, rows, acc,
                   [&](const Item<2>& it, int, int i, int quad, const floatx4_t& v0, const floatx4_t& v1)
                       __attribute__((always_inline)) { emit(it, i, quad, v0, v1); });
      });
}

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// LDS is dynamic in all of these kernels.
template <auto KERNEL, class Args>
hipError_t launch_lds(dim3 grid, int lds, hipStream_t stream, const Args& a) {
  static const hipError_t attr_err =
      hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (attr_err != hipSuccess) return attr_err;
  return launch_k(false, KERNEL, grid, dim3(kThreads), lds, stream, a);
}

}  // namespace decode
}  // namespace ttamd
