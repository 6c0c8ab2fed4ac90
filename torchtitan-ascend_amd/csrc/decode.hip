// The MoE layer for a few tokens on MI355X (gfx950).
//
//   z[t, e] = bf16(sum_d x[t, d] w_r[e, d]), the sum in 64 bits; the selection from
//   z is router_group.hip's
//   (g, u)  = w13[e] x[t]   (times the score when it is applied first)
//   a[s]    = silu(min(g, L)) * clamp(u, -L, L)              slot s = t K + k
//   out[t]  = sum_k score[s] w2[e_s] a[s]  (+ gate[t] * shared expert of x[t])
//
// Four launches, three for one token:
//   router_logits_kernel  a workgroup per row of the gate and up to 4 tokens
//   decode_plan_kernel    one workgroup: the selection, and which slots each hit
//                         expert has (for given picks only that); for one token the
//                         next two do it themselves (select_w13_kernel, plan_one)
//   stream_w13_kernel     persistent workgroups over (hit expert, row pairs)
//   stream_w2_kernel      a workgroup owns output rows, for every hit expert
// The streams: decode_stream.h.  With 4-bit weights and more than a few rows per
// expert the last two are lock_w13_kernel and lock_w2_kernel, and sum_rows_kernel
// adds the slots.  No kernel waits for another workgroup; every sum has its order, so
// a call gives the same bits every time.  Labels outside [0, E) name no expert and add
// nothing.
// Measured, experts of 1536 x 2048 and 2048 x 768, 8 picks: one token 3.2 + 15 + 8 us
// (bf16; 50 and 25 MB: each kernel's start and end are 3 to 4 us of it), 32 tokens of
// 128 experts 6 + 7 + 118 + 60 us (5.9 TB/s); in 4 bits 3 + 11 + 6 and, with the sums,
// 6 + 7 + 49 + 27 + 5.  Loads in flight bound all but the lock step (decode_stream.h).
#include <algorithm>

#include "decode_stream.h"
#include "kernels.h"
#include "router_select.h"

namespace ttamd {
namespace {

using namespace decode;

constexpr int kMaxSlots = kDecodeMaxTokens * kDecodeMaxTopk;
constexpr int kMaxE = 1024;

struct DecodeArgs {
  int T, D, H, E, K, Hs;
  const bf16_t* x;      // [T, D]
  int before;           // the score multiplies the first product
  float limit;          // NaN: none
  Weights w13, w2, s13, s2;
  bf16_t* a;            // [T K, H], then [T, Hs]
  float* y;             // lock_w2_kernel: [T K (+ T), D]
  bf16_t* out;          // [T, D]
  const char* plan;     // null (one token): made by each workgroup from the picks
  int plan_lds;         // its bytes in LDS
  const void* idx;      // one token: its picks and weights, the shared expert's factor
  const float *scores, *gate;
  int is64, split[2];   // log2 of KS: w13, w2
};

// silu(min(gate, L)) * clamp(up, -L, L) in bf16: rounded for the matrix cores, the
// only rounding between x and the output.
__device__ __forceinline__ u32x2_t activate(const floatx4_t& g, const floatx4_t& u, float limit) {
  float o[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    float gate = g[v], up = u[v];
    if (limit == limit) gate = clamp_max_nan(gate, limit), up = clamp_nan(up, limit);
    o[v] = silu_f(gate) * up;
  }
  return u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
}

// ---------------------------------------------------------------------------
// The plan: which experts are hit, and by which slots
// ---------------------------------------------------------------------------
// One workgroup makes it (with the selection, where the router runs), the two
// streaming kernels copy it to LDS.  Hit experts in order; slots sorted by expert
// ("places").
struct PlanMap {
  int T, S;
  // at 0: hit, the splits
  __host__ __device__ constexpr int valid() const { return 16; }  // uint32 [T]: which choices name an expert
  __host__ __device__ constexpr int gate() const { return valid() + 4 * T; }      // float [T]: factor of the shared one
  __host__ __device__ constexpr int score() const { return gate() + 4 * T; }      // float [S], by place
  __host__ __device__ constexpr int sorted() const { return score() + 4 * S; }    // short [S]: slot at a place
  __host__ __device__ constexpr int inverse() const { return sorted() + 2 * S; }  // short [S]: place of a slot
  __host__ __device__ constexpr int token() const { return inverse() + 2 * S; }   // short [S]: token at a place
  __host__ __device__ constexpr int list() const { return token() + 2 * S; }      // short [hit]: experts
  __host__ __device__ constexpr int start() const { return list() + 2 * S; }      // short [hit + 1]: first places
  __host__ __device__ constexpr int bytes() const { return (start() + 2 * (S + 1) + 15) & ~15; }
};
constexpr int kMaxPlanBytes = PlanMap{kDecodeMaxTokens, kMaxSlots}.bytes();

struct Plan : PlanMap {
  char* p;
  __device__ Plan(char* p_, int T_, int S_) : PlanMap{T_, S_}, p(p_) {}
  __device__ int& hit() const { return ((int*)p)[0]; }
  __device__ int& split(int i) const { return ((int*)p)[1 + i]; }  // log2 of KS: w13, w2
  __device__ uint32_t& valid(int i) const { return ((uint32_t*)(p + PlanMap::valid()))[i]; }
  __device__ float& gate(int i) const { return ((float*)(p + PlanMap::gate()))[i]; }
  __device__ float& score(int i) const { return ((float*)(p + PlanMap::score()))[i]; }
  __device__ short& sorted(int i) const { return ((short*)(p + PlanMap::sorted()))[i]; }
  __device__ short& inverse(int i) const { return ((short*)(p + PlanMap::inverse()))[i]; }
  __device__ short& token(int i) const { return ((short*)(p + PlanMap::token()))[i]; }
  __device__ short& list(int i) const { return ((short*)(p + PlanMap::list()))[i]; }
  __device__ short& start(int i) const { return ((short*)(p + PlanMap::start()))[i]; }
};

constexpr int kPlanThreads = 1024;

// What split_log needs beside the number of hit experts: items of an expert and of
// the shared one, waves to share them, stages of an item, largest log2.
struct Split {
  int items, shared, slots, stages, most;
};

struct PlanArgs {
  select::GroupTopkArgs topk;  // of the selection (its scores and idx are outputs)
  const void* idx;             // without it: given picks
  int is64;
  const float* scores;
  const float* gate;           // [T] or null: 1
  int T, E, K;
  char* plan;
  Split split[2];              // of the two products
};

// LPT = 0: given picks.  One thread per slot, then one per expert.  Barriers wait
// for LDS alone: the picks' stores need not land in between.
template <int LPT, int PL, int KL>
__global__ __launch_bounds__(kPlanThreads) void decode_plan_kernel(const PlanArgs a) {
  __shared__ int total[kMaxE];
  __shared__ float score[kMaxSlots];
  __shared__ short lab[kMaxSlots];
  __shared__ int wave_hit[kPlanThreads / 64], wave_rows[kPlanThreads / 64];
  const int S = a.T * a.K, tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const Plan p(a.plan, a.T, S);
  if (tid < a.E) total[tid] = 0;
  float gate = 1.f;
  if (tid < a.T && a.gate) gate = a.gate[tid];
  if constexpr (LPT > 0) {
    constexpr int TPB = kPlanThreads / LPT;
    const int gi = tid & (LPT - 1);
    for (int t0 = 0; t0 < a.T; t0 += TPB) {
      const int t = t0 + tid / LPT;
      if (t0 + ((tid & ~63) / LPT) >= a.T) break;  // no token for this wave
      int pick;
      double weight;
      select::select_token<LPT, PL, KL, select::SRC_BF16>(a.topk, min(t, a.T - 1), t < a.T, pick, weight, [](int) {});
      if (gi < a.K && t < a.T) {
        const float sc = (float)(weight * (double)a.topk.route_scale);
        a.topk.scores[t * a.K + gi] = score[t * a.K + gi] = sc;
        a.topk.idx[t * a.K + gi] = pick;
        lab[t * a.K + gi] = (short)pick;
      }
    }
  } else if (tid < S) {  // (S <= kPlanThreads)
    const int64_t v = a.is64 ? ((const int64_t*)a.idx)[tid] : (int64_t)((const int*)a.idx)[tid];
    lab[tid] = v >= 0 && v < a.E ? (short)v : (short)-1;
    score[tid] = a.scores[tid];
  }
  dma::lds_barrier();
  const int mine = tid < S ? lab[tid] : -1;
  int pos = 0;
  if (mine >= 0) pos = atomicAdd(&total[mine], 1);  // (columns of a product: any order gives the same sums)
  if (tid < a.T) {
    uint32_t m = (1u << a.K) - 1;
    if (LPT == 0)
      for (int k = 0; k < a.K; ++k) m &= ~((lab[tid * a.K + k] < 0 ? 1u : 0u) << k);
    p.valid(tid) = m;
    p.gate(tid) = gate;
  }
  dma::lds_barrier();
  const int n = tid < a.E ? total[tid] : 0, upto = wave_inclusive_scan(n);
  const uint64_t m = ballot64(n > 0);
  if (l == 63) wave_hit[w] = __popcll(m), wave_rows[w] = upto;
  dma::lds_barrier();
  int hit = 0, base = 0, hits = 0;
#pragma unroll
  for (int v = 0; v < kPlanThreads / 64; ++v) {
    const int h = wave_hit[v], r = wave_rows[v];
    if (v < w) hit += h, base += r;
    hits += h;
  }
  if (n > 0) {
    const int j = hit + __popcll(m & lanemask_lt()), first = base + upto - n;
    p.list(j) = (short)tid;
    p.start(j) = (short)first;
    if (j == hits - 1) p.start(hits) = (short)(first + n);
    total[tid] = first;
  }
  if (tid == kPlanThreads - 1) p.hit() = hits;
  if (l == 0 && w >= kPlanThreads / 64 - 2) {  // (waves with little else to do)
    const Split& sp = a.split[w - (kPlanThreads / 64 - 2)];
    p.split(w - (kPlanThreads / 64 - 2)) = split_log(hits * sp.items + sp.shared, sp.slots, sp.stages, sp.most);
  }
  dma::lds_barrier();
  if (mine >= 0) {
    const int at = total[mine] + pos;
    p.sorted(at) = (short)tid;
    p.token(at) = (short)(tid / a.K);
    p.inverse(tid) = (short)at;
    p.score(at) = score[tid];
  }
}

// One token needs no sorting: each of its slots is a run, in order (a repeated pick
// streams its expert again).  The first wave's lane k has choice k.
__device__ __forceinline__ void plan_one(const DecodeArgs& a, char* smem, int64_t pick, float score) {
  const Plan p(smem, 1, a.K);
  const int k = threadIdx.x;
  const bool ok = k < a.K && pick >= 0 && pick < a.E;
  const uint64_t m = ballot64(ok);
  if (ok) {
    const int j = __popcll(m & lanemask_lt());
    p.list(j) = (short)pick;
    p.score(j) = score;
    p.start(j) = (short)j;
    p.sorted(j) = (short)k;
    p.token(j) = 0;
    p.inverse(k) = (short)j;
  }
  if (k == 0) {
    const int hits = __popcll(m);
    p.hit() = hits;
    p.start(hits) = (short)hits;
    p.valid(0) = (uint32_t)m;
    p.gate(0) = a.gate ? a.gate[0] : 1.f;
    p.split(0) = a.split[0], p.split(1) = a.split[1];
  }
}

// The plan in LDS.
__device__ __forceinline__ void load_plan(const DecodeArgs& a, char* smem) {
  if (!a.plan) {
    if (threadIdx.x < 64) {
      const int k = min((int)threadIdx.x, a.K - 1);
      plan_one(a, smem, a.is64 ? ((const int64_t*)a.idx)[k] : (int64_t)((const int*)a.idx)[k], a.scores[k]);
    }
  } else {
    const int n = PlanMap{a.T, a.T * a.K}.bytes() / 16;
    for (int i = threadIdx.x; i < n; i += kThreads) ((uint4*)smem)[i] = ((const uint4*)a.plan)[i];
  }
  __syncthreads();
}

// c ? x : y by value.  (A branch would become one between the members' addresses: the
// kernel's arguments loaded again for every item, or copied to scratch.)
__device__ __forceinline__ int either(bool c, int x, int y) { return y ^ ((x ^ y) & -(int)c); }
__device__ __forceinline__ Weights either(bool c, const Weights& x, const Weights& y) {
  const uint64_t m = c ? ~0ull : 0ull;
  auto one = [&](const void* p, const void* q) {
    return (const void*)((uint64_t)q ^ (((uint64_t)p ^ (uint64_t)q) & m));
  };
  return {one(x.w, y.w), (const uint8_t*)one(x.exps, y.exps)};
}

// The hit expert at j and its rows, or the shared one: one round of LDS reads, not
// one per branch (an item of a few stages waits for them; 32 tokens of 128 experts'
// w2 of 2048 x 768 in 4 bits: 45 -> 41 us).
struct Run {
  int e, start, cnt;
};
__device__ __forceinline__ Run run_of(const DecodeArgs& a, const Plan& p, bool shared, int j) {
  j = shared ? 0 : j;
  const int e = __builtin_amdgcn_readfirstlane(p.list(j)), first = __builtin_amdgcn_readfirstlane(p.start(j)),
            end = __builtin_amdgcn_readfirstlane(p.start(j + 1));
  return {shared ? 0 : e, shared ? -1 : first, shared ? a.T : end - first};
}

// w13's items: R row pairs (gate and up rows of the same 16 hidden units) of an
// expert; wave r of them takes pair rb R + r.  The shared expert's, which have the
// most rows, come first, or in lock step last, where a last round that is not full is
// split finer.
template <int WT, int BL, bool LAST = false>
struct W13 {
  const DecodeArgs& a;
  const Plan& p;
  int R, nsh, nrb, sh0;
  __device__ W13(const DecodeArgs& a_, const Plan& p_, int R_)
      : a(a_), p(p_), R(R_), nsh((a_.Hs / 16 + R_ - 1) / R_), nrb((a_.H / 16 + R_ - 1) / R_) {
    sh0 = LAST ? __builtin_amdgcn_readfirstlane(p.hit()) * nrb : 0;
  }
  __device__ __forceinline__ int items(int hit) const { return nsh + hit * nrb; }
  __device__ __forceinline__ Item<BL> operator()(int i, int r) const {
    Item<BL> c;
    const bool shared = LAST ? i >= sh0 : i < nsh;
    const int r0 = LAST ? i : i - nsh;
    const int j = shared ? 0 : r0 / nrb;
    const Run run = run_of(a, p, shared, j);
    const int e = run.e, H = either(shared, a.Hs, a.H);
    c.rb = shared ? i - sh0 : r0 - j * nrb;
    c.start = run.start;
    c.lo = 0;
    c.cnt = run.cnt;
    c.K = a.D;
    c.x = (uint64_t)a.x;
    c.pair = r;
    const int g = c.rb * R + r;
    c.live = g < H / 16;
    const Weights m = either(shared, a.s13, a.w13);
#pragma unroll
    for (int b = 0; b < BL; ++b)
      set_load<WT>(c, b, m, e, 2 * H, a.D,
                   (b < BL / 2 ? 0 : H) + 16 * (c.live ? g : 0) + (WT == W_BF16 ? 8 * (b & 1) : 0));
    return c;
  }
  __device__ __forceinline__ uint32_t src(const Item<BL>& c, int i) const {
    const int t = p.token(max(c.start, 0) + i);  // (in the plan; the shared expert's rows are the tokens)
    return (uint32_t)(c.start < 0 ? i : t) * (uint32_t)a.D * 2u;
  }
  __device__ __forceinline__ void emit(const Item<BL>& c, int pair, int i, int quad, const floatx4_t& v0,
                                       const floatx4_t& v1) const {
    const bool shared = c.start < 0;
    const int H = shared ? a.Hs : a.H, group = c.rb * R + pair;
    if (group >= H / 16) return;
    const int slot = shared ? i : p.sorted(c.start + i);
    const float sc = shared || !a.before ? 1.f : p.score(c.start + i);
    bf16_t* const dst = a.a + (shared ? (int64_t)(a.T * a.K) * a.H : 0) + (uint32_t)slot * (uint32_t)H;
    *(u32x2_t*)(dst + 16 * group + 4 * quad) = activate(v0 * sc, v1 * sc, a.limit);
  }
};

// gate and up rows of 16 hidden units
template <int WT>
constexpr int kPairLoads = WT == W_BF16 ? 4 : 2;

constexpr int kMeetRows = 4;  // (the rings leave room for no more)

template <int WT, int NB, int NS>
__device__ __forceinline__ void stream_w13(const DecodeArgs& a, char* smem) {
  constexpr int BL = kPairLoads<WT>;
  using Rg = Ring<WT, BL, NB, NS>;
  const Plan p(smem, a.T, a.T * a.K);
  char* const ring = smem + a.plan_lds;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int log_ks = __builtin_amdgcn_readfirstlane(p.split(0)), KS = 1 << log_ks;
  const W13<WT, BL> items(a, p, kWaves >> log_ks);
  int turn = 0;
  stream_items<WT, BL, NB, NS>(
      ring, blockIdx.x, gridDim.x, items.items(__builtin_amdgcn_readfirstlane(p.hit())), w & (KS - 1), KS,
      [&](int i) __attribute__((always_inline)) { return items(i, w >> log_ks); },
      [](const Item<BL>& c, int) { return c.x; },
      [&](const Item<BL>& c, int, int i) __attribute__((always_inline)) { return items.src(c, i); },
      [&](const Item<BL>& c, int c0, int rows, const floatx4_t (&acc)[2][Rg::NT]) __attribute__((always_inline)) {
        meet_pairs<kMeetRows>(ring + Rg::kAll, turn, log_ks, c, c0, rows, acc,
                   [&](const Item<BL>& it, int r, int i, int quad, const floatx4_t& v0, const floatx4_t& v1)
                       __attribute__((always_inline)) { items.emit(it, r, i, quad, v0, v1); });
      });
}

template <int WT, int NB, int NS>
__global__ __launch_bounds__(kThreads, 2) void stream_w13_kernel(const DecodeArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  load_plan(a, smem);
  stream_w13<WT, NB, NS>(a, smem);
}

// One token: every workgroup makes the selection for itself (the first wave; equal
// bits in all), which costs it 2 to 3 us; a launch for it cost 6.5.
struct SelectArgs {
  DecodeArgs d;
  select::GroupTopkArgs topk;
};
constexpr int kSelectPerLane = 4, kSelectK = 8;  // experts of a lane, picks

template <int WT, int NB, int NS>
__global__ __launch_bounds__(kThreads, 2) void select_w13_kernel(const SelectArgs s) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int k = threadIdx.x;
  if (k < 64) {
    int pick;
    double weight;
    select::select_token<64, kSelectPerLane, kSelectK, select::SRC_BF16>(s.topk, 0, true, pick, weight, [](int) {});
    const float score = (float)(weight * (double)s.topk.route_scale);
    plan_one(s.d, smem, pick, score);
    if (blockIdx.x == 0 && k < s.d.K) {
      s.topk.scores[k] = score;
      s.topk.idx[k] = pick;
    }
  }
  __syncthreads();
  stream_w13<WT, NB, NS>(s.d, smem);
}

// More rows per expert, 4 bits.
template <int NR, int NS>
__global__ __launch_bounds__(kThreads, 2) void lock_w13_kernel(const DecodeArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const Plan p(smem, a.T, a.T * a.K);
  load_plan(a, smem);
  const W13<W_FP4, 2, true> items(a, p, kWaves);
  lock_items<NR, NS>(
      smem + a.plan_lds, items.items(__builtin_amdgcn_readfirstlane(p.hit())), (a.D + 127) / 128,
      [&](int i, int r) __attribute__((always_inline)) { return items(i, r); },
      [](const Item<2>& c, int) { return c.x; },
      [&](const Item<2>& c, int, int i) __attribute__((always_inline)) { return items.src(c, i); },
      [&](const Item<2>& c, int i, int quad, const floatx4_t& v0, const floatx4_t& v1) __attribute__((always_inline)) {
        items.emit(c, c.pair, i, quad, v0, v1);
      });
}

// A workgroup owns the output rows of BL loads (8 each, 4 bits: 16) for every
// expert; its waves (KS to a share of the columns) take the hit experts in turn, the
// weighted rows of all slots meet in LDS and leave as the tokens' sums: nothing goes
// through memory, no workgroup waits for another, every sum has its order.
template <int WT, int BL, int NB, int NS>
__global__ __launch_bounds__(kThreads, 2) void stream_w2_kernel(const DecodeArgs a) {
  using Rg = Ring<WT, BL, NB, NS>;
  constexpr int MB = Rg::kBlocks, LR = load_rows(WT);
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int S = a.T * a.K, tid = threadIdx.x, l = tid & 63;
  const Plan p(smem, a.T, S);
  char* const ring = smem + a.plan_lds;
  floatx4_t* const sums = (floatx4_t*)(ring + Rg::kAll);  // [KS][place][MB][4]
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  load_plan(a, smem);
  const int hit = __builtin_amdgcn_readfirstlane(p.hit());
  const int nsh = a.Hs > 0, places = S + (nsh ? a.T : 0);
  const int log_ks = __builtin_amdgcn_readfirstlane(p.split(1));
  const int KS = 1 << log_ks, R = kWaves >> log_ks, ks = w & (KS - 1);
  const int row0 = blockIdx.x * BL * LR;
  auto item_of = [&](int i) {
    Item<BL> c;
    const bool shared = i < nsh;
    const Run run = run_of(a, p, shared, i - nsh);
    c.rb = 0;
    c.start = run.start;
    c.lo = 0;
    c.cnt = run.cnt;
    c.K = either(shared, a.Hs, a.H);
    c.x = (uint64_t)(shared ? a.a + (int64_t)S * a.H : a.a);
    c.live = true;
#pragma unroll
    for (int b = 0; b < BL; ++b)  // (rows past the last: the last ones again, not stored)
      set_load<WT>(c, b, either(shared, a.s2, a.w2), run.e, a.D, c.K, min(row0 + b * LR, a.D - LR));
    return c;
  };
  stream_items<WT, BL, NB, NS>(
      ring, w >> log_ks, R, nsh + hit, ks, KS, item_of, [](const Item<BL>& c, int) { return c.x; },
      [&](const Item<BL>& c, int, int i) {
        const int slot = p.sorted(max(c.start, 0) + i);
        return (uint32_t)(c.start < 0 ? i : slot) * (uint32_t)c.K * 2u;
      },
      [&](const Item<BL>& c, int c0, int rows, const floatx4_t (&acc)[MB][Rg::NT]) {
#pragma unroll
        for (int t = 0; t < Rg::NT; ++t) {
          const int i = 16 * t + (l & 15);
          if (i < rows) {
            const int place = (c.start < 0 ? S : c.start) + c0 + i;
#pragma unroll
            for (int b = 0; b < MB; ++b) sums[((ks * places + place) * MB + b) * 4 + (l >> 4)] = acc[b][t];
          }
        }
      });
  __syncthreads();
  constexpr int quads = BL * LR / 4, room = 4 * MB;
  for (int i = tid; i < a.T * quads; i += kThreads) {
    const int t = i / quads, d = i % quads;
    if (row0 + 4 * d >= a.D) continue;
    auto row = [&](int place) {  // the KS shares in order
      floatx4_t v = sums[place * room + d];
      for (int j = 1; j < KS; ++j) v += sums[(j * places + place) * room + d];
      return v;
    };
    const uint32_t ok = p.valid(t);
    floatx4_t sum = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < a.K; k0 += 8) {
      bool in[8];
      int place[8];  // (reads without branches, at place 0 for no expert: one wait for all)
      float sc[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int inv = p.inverse(t * a.K + min(k0 + k, a.K - 1));
        in[k] = k0 + k < a.K && (ok >> (k0 + k) & 1);
        place[k] = in[k] ? inv : 0;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sc[k] = p.score(place[k]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const floatx4_t next = sum + row(place[k]) * (a.before ? 1.f : sc[k]);
        sum = in[k] ? next : sum;
      }
    }
    if (nsh) sum += row(S + t) * p.gate(t);
    *(u32x2_t*)(a.out + (int64_t)t * a.D + row0 + 4 * d) =
        u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
  }
}

// More rows per expert, 4 bits: the slots' weighted rows go to memory in fp32 (their
// sums would not fit the LDS beside the stages), sum_rows_kernel adds them.
template <int NR, int NS>
__global__ __launch_bounds__(kThreads, 2) void lock_w2_kernel(const DecodeArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int S = a.T * a.K;
  const Plan p(smem, a.T, S);
  load_plan(a, smem);
  const int nrb = (a.D / 32 + kWaves - 1) / kWaves, nsh = a.Hs > 0 ? nrb : 0;
  lock_items<NR, NS>(
      smem + a.plan_lds, nsh + __builtin_amdgcn_readfirstlane(p.hit()) * nrb, (a.H + 127) / 128,
      [&](int i, int r) __attribute__((always_inline)) {
        Item<2> c;
        const bool shared = i < nsh;
        const int j = shared ? 0 : (i - nsh) / nrb;
        const Run run = run_of(a, p, shared, j);
        c.rb = shared ? i : i - nsh - j * nrb;
        c.start = run.start;
        c.lo = 0;
        c.cnt = run.cnt;
        c.K = either(shared, a.Hs, a.H);
        c.x = (uint64_t)(shared ? a.a + (int64_t)S * a.H : a.a);
        c.pair = r;
        const int g = c.rb * kWaves + r;
        c.live = g < a.D / 32;
#pragma unroll
        for (int b = 0; b < 2; ++b)
          set_load<W_FP4>(c, b, either(shared, a.s2, a.w2), run.e, a.D, c.K, c.live ? 32 * g + 16 * b : 0);
        return c;
      },
      [](const Item<2>& c, int) { return c.x; },
      [&](const Item<2>& c, int, int i) {
        const int slot = p.sorted(max(c.start, 0) + i);
        return (uint32_t)(c.start < 0 ? i : slot) * (uint32_t)c.K * 2u;
      },
      [&](const Item<2>& c, int i, int quad, const floatx4_t& v0, const floatx4_t& v1) __attribute__((always_inline)) {
        const bool shared = c.start < 0;
        const int slot = shared ? S + i : p.sorted(c.start + i);
        const float sc = shared ? p.gate(i) : a.before ? 1.f : p.score(c.start + i);
        float* y = a.y + (int64_t)slot * a.D + 32 * (c.rb * kWaves + c.pair) + 4 * quad;
        *(floatx4_t*)y = v0 * sc;
        *(floatx4_t*)(y + 16) = v1 * sc;
      });
}

// out[t] = the token's rows in k order, then the shared expert's.
__global__ __launch_bounds__(256) void sum_rows_kernel(const DecodeArgs a) {
  const int quads = a.D / 4, S = a.T * a.K;
  const Plan p((char*)a.plan, a.T, S);
  for (int i = blockIdx.x * 256 + threadIdx.x; i < a.T * quads; i += gridDim.x * 256) {
    const int t = i / quads, d = 4 * (i - t * quads);
    const uint32_t ok = p.valid(t);
    const float* y = a.y + (int64_t)t * a.K * a.D + d;
    floatx4_t sum = {0.f, 0.f, 0.f, 0.f}, sh = sum;
    if (a.Hs > 0) sh = *(const floatx4_t*)(a.y + (int64_t)(S + t) * a.D + d);
    for (int k0 = 0; k0 < a.K; k0 += 8) {
      floatx4_t v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)  // (rows of no expert hold nothing; they are not added)
        if (k0 + k < a.K) v[k] = *(const floatx4_t*)(y + (int64_t)(k0 + k) * a.D);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < a.K && (ok >> (k0 + k) & 1)) sum += v[k];
    }
    sum += sh;
    *(u32x2_t*)(a.out + (int64_t)t * a.D + d) = u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
  }
}

// z[t, e] = bf16(sum_d x[t, d] w[e, d]).  Products of bf16 pairs are exact in 64
// bits and so are nearly all their sums, so a logit does not depend on the order
// of its terms and equal inputs give equal picks in every batch.  Row E: the
// shared expert's gate, through a sigmoid.  Bound by latency: a workgroup takes one row
// and TB tokens, its four waves every fourth 512 columns, kAhead steps' loads at a
// time (64 tokens x 33 rows of 7168: a wave per row 12.9 us, so 7.4).
constexpr int kAhead = 4;
template <int TB>
__global__ __launch_bounds__(256) void router_logits_kernel(const bf16_t* __restrict__ x,
                                                            const bf16_t* __restrict__ w_router,
                                                            const bf16_t* __restrict__ w_gate, int T, int E, int D,
                                                            bf16_t* __restrict__ logits, float* __restrict__ gate) {
  __shared__ double part[4][TB];
  const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e = blockIdx.x, t0 = blockIdx.y * TB;
  const bf16_t* w = e < E ? w_router + (int64_t)e * D : w_gate;
  double acc[TB];
#pragma unroll
  for (int t = 0; t < TB; ++t) acc[t] = 0.0;
  for (int k0 = 8 * (int)threadIdx.x; k0 < D; k0 += 2048 * kAhead) {
    uint4 wv[kAhead], xv[kAhead][TB];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k = min(k0 + 2048 * j, D - 8);
      wv[j] = *(const uint4*)(w + k);
#pragma unroll
      for (int t = 0; t < TB; ++t) xv[j][t] = *(const uint4*)(x + (int64_t)min(t0 + t, T - 1) * D + k);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (k0 + 2048 * j >= D) break;
      float wf[8], xf[8];
      unpack8(wv[j], wf);
#pragma unroll
      for (int t = 0; t < TB; ++t) {
        unpack8(xv[j][t], xf);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[t] = __builtin_fma((double)xf[i], (double)wf[i], acc[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TB; ++t) {
    double v = acc[t];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if (l == 0) part[wave][t] = v;
  }
  __syncthreads();
  const int t = threadIdx.x;
  if (t < TB && t0 + t < T) {
    const uint32_t z = f32_to_bf16((float)(((part[0][t] + part[1][t]) + part[2][t]) + part[3][t]));
    if (e < E) logits[(int64_t)(t0 + t) * E + e] = (bf16_t)z;
    else gate[t0 + t] = 1.f / (1.f + expf(-bf16_to_f32(z)));
  }
}

size_t al256(size_t n) { return (n + 255) & ~(size_t)255; }

// A call's kernels, chosen before the plan is made (it takes their splits).
struct Choice {
  hipError_t (*w13)(const DecodeArgs&, hipStream_t);
  hipError_t (*select_w13)(const SelectArgs&, hipStream_t);  // one token (null: not that form)
  hipError_t (*w2)(const DecodeArgs&, hipStream_t);
  Split split[2];
};

template <int WT, int NB, int NS>
hipError_t go_w13(const DecodeArgs& a, hipStream_t stream) {
  const int64_t pairs = (int64_t)std::min(a.E, a.T * a.K) * (a.H / 16) + a.Hs / 16;  // items at the finest
  return launch_lds<stream_w13_kernel<WT, NB, NS>>(
      dim3((unsigned)std::min<int64_t>(pairs, num_cus())),
      a.plan_lds + Ring<WT, kPairLoads<WT>, NB, NS>::kAll + meet_bytes(kMeetRows), stream, a);
}

template <int WT, int NB, int NS>
hipError_t go_select_w13(const SelectArgs& s, hipStream_t stream) {
  const int64_t pairs = (int64_t)s.d.K * (s.d.H / 16) + s.d.Hs / 16;
  return launch_lds<select_w13_kernel<WT, NB, NS>>(
      dim3((unsigned)std::min<int64_t>(pairs, num_cus())),
      s.d.plan_lds + Ring<WT, kPairLoads<WT>, NB, NS>::kAll + meet_bytes(kMeetRows), stream, s);
}

template <int WT, int NB, int NS>
bool use_w13(const DecodeArgs& a, Choice& c) {
  using Rg = Ring<WT, kPairLoads<WT>, NB, NS>;
  if (a.plan_lds + Rg::kAll + meet_bytes(kMeetRows) > kLds) return false;
  const int64_t pairs = (int64_t)std::min(a.E, a.T * a.K) * (a.H / 16) + a.Hs / 16;
  c.w13 = go_w13<WT, NB, NS>;
  if constexpr (NB == 1 && NS == (WT == W_BF16 ? 3 : 5)) c.select_w13 = go_select_w13<WT, NB, NS>;
  c.split[0] = {a.H / 16, a.Hs / 16, kWaves * (int)std::min<int64_t>(pairs, num_cus()), ceil_div(a.D, Rg::kCols), 3};
  return true;
}

template <int WT, int BL, int NB, int NS>
int w2_log(const DecodeArgs& a) {  // the most waves that may share an item (log2), -1: no room for the sums
  using Rg = Ring<WT, BL, NB, NS>;
  const int base = a.plan_lds + Rg::kAll;
  const int sums = (a.T * a.K + (a.Hs > 0 ? a.T : 0)) * Rg::kBlocks * 64;
  int most = -1;
  while (most < 3 && base + (sums << (most + 1)) <= kLds) ++most;
  return most;
}

template <int WT, int BL, int NB, int NS>
hipError_t go_w2(const DecodeArgs& a, hipStream_t stream) {
  using Rg = Ring<WT, BL, NB, NS>;
  const int sums = (a.T * a.K + (a.Hs > 0 ? a.T : 0)) * Rg::kBlocks * 64;
  return launch_lds<stream_w2_kernel<WT, BL, NB, NS>>(dim3(ceil_div(a.D, BL * load_rows(WT))),
                                                      a.plan_lds + Rg::kAll + (sums << w2_log<WT, BL, NB, NS>(a)),
                                                      stream, a);
}

template <int WT, int BL, int NB, int NS>
bool use_w2(const DecodeArgs& a, Choice& c) {
  const int most = w2_log<WT, BL, NB, NS>(a);
  if (most < 0) return false;
  c.w2 = go_w2<WT, BL, NB, NS>;
  c.split[1] = {1, a.Hs > 0, kWaves, ceil_div(std::max(a.H, a.Hs), Ring<WT, BL, NB, NS>::kCols), most};
  return true;
}

// bf16.  Token rows per pass by the rows that an expert gets on average (up to 8
// tokens fit one pass of 8 anyway): a pass more streams its weights again, a larger one
// takes LDS from the ring.  The second product takes as few output rows per workgroup as
// give one workgroup per CU at most, where the slots' sums leave the room.
// Both sides (the stage of 8 picks from 32 experts of 1536 x 2048, captured, us; the
// other product as chosen):
//   w13, 8 / 16 rows a pass    average 4: 70 / 70, 5: 91 / 74
//   w13, 16 / 32               average 10: 78 / 80, 12: 100 / 85
//   w2, 8 / 16                 average 4: 71 / 71, 5: 74 / 74, 8: 85 / 76
//   w2, 16 / 32                average 10: 81 / 84, 12: 86 / 85, 16: 89 / 84
// The average counts the routed experts: a shared one of more tokens than a pass holds
// is streamed again for every pass (16 experts of 5120 x 8192, one pick and a shared one
// as wide: 32 tokens 827 us, 526 without it).
template <int BL>
bool use_w2_bf16(const DecodeArgs& a, int rows, Choice& c) {
  if (rows <= 4)
    return use_w2<W_BF16, BL, 1, BL == 1 ? 7 : BL == 2 ? 5 : 3>(a, c) ||
           use_w2<W_BF16, BL, 1, BL == 1 ? 4 : BL == 2 ? 3 : 2>(a, c);
  if (rows <= 10)
    return use_w2<W_BF16, BL, 2, BL == 1 ? 5 : BL == 2 ? 4 : 2>(a, c) || use_w2<W_BF16, BL, 2, 2>(a, c);
  if constexpr (BL <= 2) return use_w2<W_BF16, BL, 4, 2>(a, c);
  return false;
}

bool choose_bf16(const DecodeArgs& a, Choice& c) {
  const int rows = a.T <= 8 ? 1 : ceil_div(a.T * a.K, a.E);
  const bool first = rows <= 2   ? use_w13<W_BF16, 1, 3>(a, c)
                     : rows <= 8 ? use_w13<W_BF16, 2, 3>(a, c) || use_w13<W_BF16, 2, 2>(a, c)
                                  : use_w13<W_BF16, 4, 2>(a, c);
  const int loads = ceil_div(a.D, 8 * num_cus());
  return first && ((loads <= 1 && use_w2_bf16<1>(a, rows, c)) || (loads <= 2 && use_w2_bf16<2>(a, rows, c)) ||
                   (loads <= 3 && use_w2_bf16<3>(a, rows, c)) || use_w2_bf16<4>(a, rows, c) ||
                   use_w2<W_BF16, 2, 4, 2>(a, c) || use_w2<W_BF16, 2, 1, 2>(a, c));
}

template <int NR, int NS>
hipError_t go_lock_w13(const DecodeArgs& a, hipStream_t stream) {
  const int64_t items = (int64_t)std::min(a.E, a.T * a.K) * ceil_div(a.H / 16, kWaves) + ceil_div(a.Hs / 16, kWaves);
  return launch_lds<lock_w13_kernel<NR, NS>>(dim3((unsigned)std::min<int64_t>(items, num_cus())),
                                             a.plan_lds + Lock<NR, NS>::kAll, stream, a);
}
template <int NR, int NS>
hipError_t go_lock_w2(const DecodeArgs& a, hipStream_t stream) {
  const int64_t items = (int64_t)(std::min(a.E, a.T * a.K) + (a.Hs > 0)) * ceil_div(a.D / 32, kWaves);
  const hipError_t err =
      launch_lds<lock_w2_kernel<NR, NS>>(dim3((unsigned)std::min<int64_t>(items, num_cus())),
                                         a.plan_lds + Lock<NR, NS>::kAll, stream, a);
  if (err != hipSuccess) return err;
  return launch_k(false, sum_rows_kernel, dim3(std::min(ceil_div(a.T * (a.D / 4), 256), 4 * num_cus())), dim3(256), 0,
                  stream, a);
}

// 4 bits.  A stream's token rows take as much LDS as its weights: for few rows per
// expert (up to 4 tokens fit one pass of 4), else all waves of a workgroup share them, as
// they do for a shared expert of many tokens.  Both sides, streams / lock step (8 picks,
// captured, us): 32 experts of 1536 x 2048, average 4: 36 / 39, 5: 45 / 39; 4096 x 7168, 4:
// 148 / 162, 6: 171 / 164; with a shared expert, 16 tokens 169 / 170, 20 186 / 170 (128 of
// 1536 x 2048: 12 tokens 68 / 64, 16 76 / 71, 20 86 / 80).
bool choose_fp4(const DecodeArgs& a, Choice& c) {
  const int64_t S = (int64_t)a.T * a.K;
  const int rows = a.T <= 4 ? 1 : ceil_div(S, a.E);
  if (rows > 4 || (a.Hs > 0 && a.T > 16)) {
    c.w13 = go_lock_w13<1, 5>;
    c.w2 = go_lock_w2<1, 5>;
    static_assert(((kMaxPlanBytes + 127) & ~127) + Lock<1, 5>::kAll <= kLds, "LDS");
    return true;
  }
  // The second product's workgroups own 16 output rows, or 32 where 16 would make more
  // of them than the chip has CUs, or 8 where 16 would leave half of it idle (2048 rows of
  // 768: one token's 8 experts 7.3 us by 16, 6.3 by 8; 8 tokens' 50 experts 30 and 21).
  const int blocks = a.D / 16, cus = num_cus();
  // lock_w2_kernel and its sums instead where items are a few stages, so that a stream
  // waits for the plan more than for weights, and slots enough to pay for the launch (32
  // tokens of 128 experts, 2048 x 768: 41 us, so 32; 8 tokens 18.9 and 19.4; 8 of 32
  // experts, 7168 x 2048: 37 and 51), and where the LDS has no room for all slots' sums
  // beside a ring (64 tokens of 128 experts: a ring of 3 stages 70 us, so 33).
  // Around these bounds (the stage, captured, streams / lock step, us): 2048 x 768, 64 slots
  // 52.5 / 51.8, 96 63.6 / 61.9, 128 68.0 / 63.3; 128 slots, H = 1024 83.6 / 79.3, H = 1280
  // 98.4 / 89.7, so that 2048 columns would gain past 1024 too; 4096 columns do not below:
  // 96 slots of 4096 x 768 89.6 / 92.2, x 1024 107.5 / 111.7.
  bool first, second;
  if (rows <= 2) {
    first = use_w13<W_FP4, 1, 5>(a, c) || use_w13<W_FP4, 1, 4>(a, c);
    second = 2 * blocks <= cus ? use_w2<W_FP4_8, 1, 2, 5>(a, c)
             : blocks <= cus   ? use_w2<W_FP4, 1, 1, 7>(a, c)
                               : use_w2<W_FP4, 2, 1, 4>(a, c);
  } else {
    first = use_w13<W_FP4, 2, 4>(a, c) || use_w13<W_FP4, 2, 3>(a, c);
    second = 2 * blocks <= cus ? use_w2<W_FP4_8, 1, 4, 3>(a, c)
             : blocks <= cus   ? use_w2<W_FP4, 1, 2, 5>(a, c)
                               : use_w2<W_FP4, 2, 2, 3>(a, c);
  }
  if (!second || (S > 64 && std::max(a.H, a.Hs) <= 1024)) c.w2 = go_lock_w2<1, 5>, c.select_w13 = nullptr;
  return first;
}

template <int LPT, int PL>
hipError_t go_plan(const PlanArgs& a, hipStream_t stream) {
  auto kernel = a.K <= 8 ? decode_plan_kernel<LPT, PL, 8> : decode_plan_kernel<LPT, PL, 16>;
  return launch_k(false, kernel, dim3(1), dim3(kPlanThreads), 0, stream, a);
}

// The selection and the plan.  A wave per token (16 at a time) while that is one
// round, else 16 lanes (64 tokens at a time) where they can hold the experts.
hipError_t launch_plan_topk(PlanArgs a, hipStream_t stream) {
  select::GroupTopkArgs& t = a.topk;
  int lr16 = 0, lr64 = 0;
  const int p16 = select::experts_per_lane(16, t.G, t.EG, &lr16), p64 = select::experts_per_lane(64, t.G, t.EG, &lr64);
  const bool narrow = p16 > 0 && p16 <= 16 && (p16 <= 4 || a.T > 16);
  t.log_run = narrow ? lr16 : lr64;
  t.per_lane = narrow ? p16 : p64;
  if (narrow) {
    if (p16 <= 4) return go_plan<16, 4>(a, stream);
    if (p16 <= 8) return go_plan<16, 8>(a, stream);
    if (p16 <= 12) return go_plan<16, 12>(a, stream);
    return go_plan<16, 16>(a, stream);
  }
  if (p64 <= 4) return go_plan<64, 4>(a, stream);
  if (p64 <= 8) return go_plan<64, 8>(a, stream);
  if (p64 <= 16) return go_plan<64, 16>(a, stream);
  return go_plan<64, 32>(a, stream);  // E <= 1024, G <= 64: at most 32 per lane
}

}  // namespace

size_t router_decode_workspace_bytes(int64_t T, int E) { return al256((size_t)T * E * 2); }

namespace {

hipError_t launch_logits(const RouterDecode& r, int T, int E, int D, hipStream_t stream) {
  const int rows = E + (r.w_gate != nullptr);
  const int tb = T >= 4 ? 4 : T >= 2 ? 2 : 1;
  const dim3 grid(rows, ceil_div(T, tb));
  auto kernel = tb == 4 ? router_logits_kernel<4> : tb == 2 ? router_logits_kernel<2> : router_logits_kernel<1>;
  return launch_k(false, kernel, grid, dim3(256), 0, stream, (const bf16_t*)r.x, (const bf16_t*)r.w_router,
                  (const bf16_t*)r.w_gate, T, E, D, (bf16_t*)r.logits, r.gate);
}

}  // namespace

hipError_t launch_router_decode(const RouterDecode& r, int T, int E, int D, int K, hipStream_t stream) {
  const hipError_t err = launch_logits(r, T, E, D, stream);
  if (err != hipSuccess) return err;
  return launch_router_topk_grouped(r.logits, true, r.bias, T, E, K, r.groups, r.score_func, r.renorm, r.eps, r.scale,
                                    r.top_scores, r.top_idx, stream);
}

// Workspace: the plan, activations of the slots and of the shared expert, their
// fp32 output rows (lock_w2_kernel's; of 4-bit weights, but one size serves both types).
size_t experts_decode_workspace_bytes(int64_t T, int64_t D, int64_t H, int K, int64_t Hs) {
  const int64_t S = T * K;
  return al256(PlanMap{(int)T, (int)S}.bytes()) + al256((size_t)(S * H + (Hs > 0 ? T * Hs : 0)) * 2) +
         al256((size_t)(S + (Hs > 0 ? T : 0)) * D * 4);
}

hipError_t launch_experts_decode(const ExpertsDecode& c, const RouterDecode* router, void* ws, hipStream_t stream) {
  DecodeArgs a{};
  a.T = c.T, a.D = c.D, a.H = c.H, a.E = c.E, a.K = c.K, a.Hs = c.Hs;
  a.x = (const bf16_t*)c.x;
  a.before = c.before, a.limit = c.limit;
  a.w13 = {c.w13, c.e13}, a.w2 = {c.w2, c.e2}, a.s13 = {c.s13, c.es13}, a.s2 = {c.s2, c.es2};
  const int64_t S = (int64_t)a.T * a.K, Ts = a.Hs > 0 ? a.T : 0;
  const PlanMap map{a.T, (int)S};
  char* p = (char*)ws;
  a.plan = p;
  a.plan_lds = (map.bytes() + 127) & ~127;
  p += al256(map.bytes());
  a.a = (bf16_t*)p;
  p += al256((size_t)(S * a.H + Ts * a.Hs) * 2);
  a.y = (float*)p;
  a.out = (bf16_t*)c.out;
  Choice choice{};
  if (!(c.fp4 ? choose_fp4(a, choice) : choose_bf16(a, choice))) return hipErrorInvalidValue;

  hipError_t err = router ? launch_logits(*router, a.T, a.E, a.D, stream) : hipSuccess;
  if (err != hipSuccess) return err;
  select::GroupTopkArgs t{};
  if (router) {
    t.z = router->logits;
    t.S = 1, t.T = a.T, t.E = a.E, t.K = a.K;
    t.aligned = ((uintptr_t)router->logits & 15) == 0;
    t.G = router->groups.groups, t.EG = a.E / t.G, t.kept = router->groups.kept, t.top2 = router->groups.top2;
    t.bias = router->bias;
    t.score_func = router->score_func, t.renorm = router->renorm, t.eps = router->eps, t.route_scale = router->scale;
    t.scores = router->top_scores, t.idx = router->top_idx;
  }
  if (a.T == 1 && choice.select_w13) {
    int log_run = 0;
    const int per_lane = router ? select::experts_per_lane(64, t.G, t.EG, &log_run) : 0;
    if (!router || (per_lane > 0 && per_lane <= kSelectPerLane && a.K <= kSelectK)) {
      a.plan = nullptr;
      a.idx = router ? (const void*)router->top_idx : c.idx, a.is64 = router || c.is64;
      a.scores = router ? router->top_scores : c.scores;
      a.gate = c.gate;
      for (int i = 0; i < 2; ++i) {
        const Split& sp = choice.split[i];
        a.split[i] = split_log(a.K * sp.items + sp.shared, sp.slots, sp.stages, sp.most);
      }
      if (router) {
        t.log_run = log_run, t.per_lane = per_lane;
        err = choice.select_w13(SelectArgs{a, t}, stream);
      } else {
        err = choice.w13(a, stream);
      }
      return err != hipSuccess ? err : choice.w2(a, stream);
    }
  }

  PlanArgs pa{};
  pa.topk = t;
  pa.idx = c.idx, pa.is64 = c.is64, pa.scores = c.scores, pa.gate = c.gate;
  pa.T = a.T, pa.E = a.E, pa.K = a.K, pa.plan = (char*)ws;
  pa.split[0] = choice.split[0], pa.split[1] = choice.split[1];
  err = router ? launch_plan_topk(pa, stream) : go_plan<0, 4>(pa, stream);
  if (err != hipSuccess) return err;
  err = choice.w13(a, stream);
  return err != hipSuccess ? err : choice.w2(a, stream);
}

}  // namespace ttamd
