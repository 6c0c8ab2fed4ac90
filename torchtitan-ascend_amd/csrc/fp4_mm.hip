// Products of a few rows with 4-bit weights on MI355X (gfx950):
// out[m] = x[m] w[e]^T (+ bias), expert e's rows offs[e - 1] .. offs[e] - 1, or all of
// them for one matrix.
//
// Bound by the weights' bytes (17/32 per value); the streams of decode_stream.h.  With
// few rows per matrix a wave streams 32 output rows by itself, or KS waves together
// where that fills the chip; with more, a workgroup's waves share the token rows.
// Measured: 1 x 5120 x 8192 9.8 us (22 MB; 160 workgroups have rows), 13 x 1000 x 1440
// 6.7, 96 rows of 68 of 128 matrices of 1536 x 2048 31.7 (114 MB, 4.5 TB/s between
// start and end).
//
// A pass's token rows are 4, 8, 16, 32 or 64, chosen on the host from the rows that a
// matrix gets on average; a matrix with more streams its weights again for every pass.
// Both sides (captured, us, about 6 of them the graph's launch):
//   grouped, 128 of 1536 x 2048    4 / 8 rows a pass, average 2: 48 / 42, 3: 61 / 48;
//                                  8 / 32, 4: 52 / 50, 5: 57 / 53; 32 / 64, 24: 71 / 65, 32:
//                                  93 / 76, 40: 102 / 78 (the hottest matrix has 1.5 times that)
//   dense, 5120 x 8192             4 / 8, 2 to 4 rows: equal; 8 / 16, 9: 19 / 17; 16 / 32 in
//                                  lock step, 16: 18 / 50, 17: 20 / 57; 16 / 64, 64: 28 / 87, 128:
//                                  46 / 87; 16384 x 2048, 17: 19 / 21, 64: 19 / 29, 128: 33 / 30
// so the lock step loses above 16 dense rows where N / 256 workgroups leave CUs idle,
// and at 24 to 32 grouped ones.  A skewed load pays for the average: 200 rows of 128
// matrices 47 us spread evenly, 197 with 96 of them on one; 4096 rows of 1024 matrices
// of 256 x 512 20 us, 536 on one.
#include <algorithm>

#include "decode_stream.h"
#include "kernels.h"

namespace ttamd {
namespace {

using namespace decode;

constexpr int kMaxE = 1024;

struct MmArgs {
  const bf16_t* x;
  Weights w;
  const int* offs;  // null: one matrix, rows in tiles of `tile`
  const void* bias;
  int bias32, M, E, N, K;
  int tile, tiles;
  bf16_t* out;
};

// The matrices that have rows, and their rows.
struct Runs {
  int n;
  int first[kMaxE], end[kMaxE];
  short list[kMaxE];
  int wave[kWaves];
};

__device__ __forceinline__ void find_runs(const MmArgs& a, Runs& s) {
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  int base = 0;
  for (int e0 = 0; e0 < a.E; e0 += kThreads) {
    const int e = e0 + tid;
    int r0 = 0, r1 = 0;
    if (e < a.E) {
      r0 = e > 0 ? min(max(a.offs[e - 1], 0), a.M) : 0;
      r1 = min(max(a.offs[e], 0), a.M);
    }
    const uint64_t m = ballot64(r1 > r0);
    if (l == 0) s.wave[w] = __popcll(m);
    __syncthreads();
    int at = base;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      if (v < w) at += s.wave[v];
      base += s.wave[v];
    }
    if (r1 > r0) {
      const int j = at + __popcll(m & lanemask_lt());
      s.list[j] = (short)e, s.first[j] = r0, s.end[j] = r1;
    }
    __syncthreads();
  }
  if (tid == 0) s.n = base;
  __syncthreads();
}

// Items: R pairs of 16-row blocks of a matrix times its rows (one matrix: a tile of
// them).
struct MmItems {
  const MmArgs& a;
  const Runs& s;
  int R, nrb;
  __device__ MmItems(const MmArgs& a_, const Runs& s_, int R_)
      : a(a_), s(s_), R(R_), nrb((((a_.N + 15) / 16 + 1) / 2 + R_ - 1) / R_) {}
  __device__ __forceinline__ int items(int runs) const { return runs * nrb; }
  __device__ __forceinline__ Item<2> operator()(int i, int r) const {
    Item<2> c;
    const int j = i / nrb;
    int e = 0;
    c.rb = i - j * nrb;
    if (a.offs) {
      e = __builtin_amdgcn_readfirstlane(s.list[j]);
      c.start = __builtin_amdgcn_readfirstlane(s.first[j]);
      c.cnt = __builtin_amdgcn_readfirstlane(s.end[j]) - c.start;
    } else {
      c.start = j * a.tile;
      c.cnt = min(a.tile, a.M - c.start);
    }
    c.lo = 0;
    c.K = a.K;
    c.x = (uint64_t)(a.x + (int64_t)c.start * a.K);
    c.pair = r;
    const int g = c.rb * R + r, blocks = (a.N + 15) / 16;
    c.live = 2 * g < blocks;
    // (a block past the last: the last again, not stored)
    set_load<W_FP4>(c, 0, a.w, e, a.N, a.K, 16 * min(2 * g, blocks - 1));
    set_load<W_FP4>(c, 1, a.w, e, a.N, a.K, 16 * min(2 * g + 1, blocks - 1));
    return c;
  }
  __device__ __forceinline__ uint64_t origin(const Item<2>& c, int n0) const {
    return c.x + (uint64_t)n0 * (uint64_t)a.K * 2;
  }
  __device__ __forceinline__ uint32_t src(int n0, int i) const { return (uint32_t)(i - n0) * (uint32_t)a.K * 2u; }
  __device__ __forceinline__ float bias(int n) const {
    return a.bias32 ? ((const float*)a.bias)[n] : bf16_to_f32(((const bf16_t*)a.bias)[n]);
  }
  __device__ __forceinline__ void store(int64_t row, int n, floatx4_t v) const {
    if (n >= a.N) return;
    const int last = a.N - 1 - n;
    if (a.bias) v += floatx4_t{bias(n), bias(n + min(1, last)), bias(n + min(2, last)), bias(n + min(3, last))};
    bf16_t* const out = a.out + row * a.N + n;
    const u32x2_t o = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    if ((a.N & 3) == 0) {
      *(u32x2_t*)out = o;
    } else {
      out[0] = (bf16_t)o[0];
      if (last >= 1) out[1] = (bf16_t)(o[0] >> 16);
      if (last >= 2) out[2] = (bf16_t)o[1];
      if (last >= 3) out[3] = (bf16_t)(o[1] >> 16);
    }
  }
  __device__ __forceinline__ void emit(const Item<2>& c, int pair, int i, int quad, const floatx4_t& v0,
                                       const floatx4_t& v1) const {
    const int n = 32 * (c.rb * R + pair) + 4 * quad;
    store(c.start + i, n, v0);
    store(c.start + i, n + 16, v1);
  }
};

constexpr int kRunsBytes = (sizeof(Runs) + 127) & ~127;

template <int NB, int NS>
__global__ __launch_bounds__(kThreads, 2) void stream_mm_kernel(const MmArgs a) {
  using Rg = Ring<W_FP4, 2, NB, NS>;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  Runs& s = *(Runs*)smem;
  char* const ring = smem + (a.offs ? kRunsBytes : 0);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int runs = a.tiles;
  if (a.offs) {
    find_runs(a, s);
    runs = __builtin_amdgcn_readfirstlane(s.n);
  }
  const int log_ks = split_log(runs * (((a.N + 15) / 16 + 1) / 2), kWaves * gridDim.x, (a.K + 127) / 128, 3);
  const int KS = 1 << log_ks;
  const MmItems items(a, s, kWaves >> log_ks);
  int turn = 0;
  stream_items<W_FP4, 2, NB, NS>(
      ring, blockIdx.x, gridDim.x, items.items(runs), w & (KS - 1), KS,
      [&](int i) __attribute__((always_inline)) { return items(i, w >> log_ks); },
      [&](const Item<2>& c, int n0) __attribute__((always_inline)) { return items.origin(c, n0); },
      [&](const Item<2>&, int n0, int i) __attribute__((always_inline)) { return items.src(n0, i); },
      [&](const Item<2>& c, int c0, int rows, const floatx4_t (&acc)[2][Rg::NT]) __attribute__((always_inline)) {
        meet_pairs<Rg::kRows>(ring + Rg::kAll, turn, log_ks, c, c0, rows, acc,
                   [&](const Item<2>& it, int r, int i, int quad, const floatx4_t& v0, const floatx4_t& v1)
                       __attribute__((always_inline)) {
                     items.emit(it, r, i, quad, v0, v1);
                   });
      });
}

template <int NR, int NS>
__global__ __launch_bounds__(kThreads, 2) void lock_mm_kernel(const MmArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  Runs& s = *(Runs*)smem;
  int runs = a.tiles;
  if (a.offs) {
    find_runs(a, s);
    runs = __builtin_amdgcn_readfirstlane(s.n);
  }
  const MmItems items(a, s, kWaves);
  lock_items<NR, NS>(
      smem + (a.offs ? kRunsBytes : 0), items.items(runs), (a.K + 127) / 128,
      [&](int i, int r) __attribute__((always_inline)) { return items(i, r); },
      [&](const Item<2>& c, int n0) __attribute__((always_inline)) { return items.origin(c, n0); },
      [&](const Item<2>&, int n0, int i) __attribute__((always_inline)) { return items.src(n0, i); },
      [&](const Item<2>& c, int i, int quad, const floatx4_t& v0, const floatx4_t& v1) __attribute__((always_inline)) {
        items.emit(c, c.pair, i, quad, v0, v1);
      });
}

template <int NB, int NS>
hipError_t go_stream(const MmArgs& a, int64_t pairs, hipStream_t stream) {
  constexpr int lds = Ring<W_FP4, 2, NB, NS>::kAll + meet_bytes(Ring<W_FP4, 2, NB, NS>::kRows);
  static_assert(lds + kRunsBytes <= kLds, "LDS");
  return launch_lds<stream_mm_kernel<NB, NS>>(dim3((unsigned)std::min<int64_t>(pairs, num_cus())),
                                              lds + (a.offs ? kRunsBytes : 0), stream, a);
}

template <int NR, int NS>
hipError_t go_lock(const MmArgs& a, int64_t pairs, hipStream_t stream) {
  constexpr int lds = Lock<NR, NS>::kAll;
  static_assert(lds + kRunsBytes <= kLds, "LDS");
  return launch_lds<lock_mm_kernel<NR, NS>>(dim3((unsigned)std::min<int64_t>((pairs + kWaves - 1) / kWaves, num_cus())),
                                            lds + (a.offs ? kRunsBytes : 0), stream, a);
}

}  // namespace

hipError_t launch_grouped_mm_fp4(const void* x, const void* codes, const void* exps, const int* offs, const void* bias,
                                 bool bias32, int M, int E, int N, int K, void* out, hipStream_t stream) {
  MmArgs a{};
  a.x = (const bf16_t*)x, a.w = {codes, (const uint8_t*)exps}, a.offs = offs, a.bias = bias, a.bias32 = bias32;
  a.M = M, a.E = E, a.N = N, a.K = K, a.out = (bf16_t*)out;
  const int64_t pairs = ceil_div(ceil_div(N, 16), 2);
  // rows of a matrix: given, or what it gets on average
  const int rows = offs ? ceil_div(M, E) : M;
  const bool few = rows <= (offs ? 4 : 16);
  a.tile = few ? 16 : rows <= 32 ? 32 : 64;
  a.tiles = ceil_div(M, a.tile);
  const int64_t all = pairs * (offs ? std::min(E, M) : a.tiles);
  if (few) return rows <= 2 ? go_stream<1, 5>(a, all, stream) : rows <= 8 ? go_stream<2, 3>(a, all, stream)
                                                                         : go_stream<4, 2>(a, all, stream);
  return rows <= 32 ? go_lock<1, 5>(a, all, stream) : go_lock<2, 4>(a, all, stream);
}

}  // namespace ttamd
