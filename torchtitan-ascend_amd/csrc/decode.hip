// The MoE layer for a few tokens on MI355X (gfx950), and products of rows with
// 4-bit weights.
//
//   z[t, e] = bf16(sum_d x[t, d] w_r[e, d]), the sum in 64 bits; the selection from
//   z is router_group.hip's
//   (g, u)  = w13[e] x[t]   (times the score when it is applied first)
//   a[s]    = silu(min(g, L)) * clamp(u, -L, L)              slot s = t K + k
//   out[t]  = sum_k score[s] w2[e_s] a[s]  (+ gate[t] * shared expert of x[t])
//
// A few tokens stream every hit expert's weights once and do almost nothing with
// them, so the kernels are a stream of weight rows through
// v_mfma_f32_16x16x32_bf16: A = 16 weight rows x 32 columns, straight from HBM into
// registers (a lane's 16 bytes are its share of the fragment; nothing goes
// through LDS), B = up to 16 tokens, from LDS, columns past the last token
// repeating it.  A wave owns a pair of 16-row blocks (gate and up rows of the same
// 16 hidden units; 32 output rows), so one B fragment serves two products, and
// KS waves of a workgroup may share a pair, each with every KS-th unit of its
// columns: with few rows in all that is what fills the chip.
//
// Three launches and the selection:
//   router_logits_kernel  one wave per expert and up to 8 tokens
//   decode_w13_kernel     one workgroup per hit expert and 8 / KS row pairs
//   decode_w2_kernel      the same; a slot's rows go to HBM in fp32, and the last
//                         workgroup to finish a run of output rows (an arrival
//                         counter) adds them over k in order: no waiting, and the
//                         same bits whichever is last
// Which experts are hit is not known on the host: each workgroup finds the j-th
// distinct label among the T K by itself (kFirst: the first slot of every expert).
// Labels outside [0, E) name no expert and add nothing.
#include <algorithm>

#include "common.h"
#include "dma_asm.h"
#include "fp4.h"
#include "gemm_common.h"
#include "kernels.h"

namespace ttamd {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxSlots = kDecodeMaxTokens * kDecodeMaxTopk;
constexpr int kMaxE = 1024;
// LDS for token rows: 64 rows of 512 columns or 16 of 2048, each 16 bytes apart
// from a multiple of 256 so that 16 rows' 16-byte reads meet no bank twice; two
// workgroups per CU with the labels.
constexpr int kRowBytes = 66560;

enum WeightType { W_BF16 = 0, W_FP4 = 1 };

// Columns per pipeline unit of a wave: 128 of bf16 (eight 1 KB loads a pair),
// 256 of 4 bits (four, and two exponent dwords).
template <int WT>
constexpr int kUnit = WT == W_BF16 ? 128 : 256;

// Weights [E, N, K]: bf16 rows, or 4-bit tiles and their exponents (fp4.hip).
struct Weights {
  const void* w;
  const uint8_t* exps;
};

// One wave's pair of row blocks, as lane addresses.
template <int WT>
struct Pair;

template <>
struct Pair<W_FP4> {
  const uint4 *p0, *p1;
  const uint32_t *x0, *x1;
  int C;
  __device__ __forceinline__ Pair(const Weights& m, int64_t e, int N, int K, int b0, int b1, int l) : C((K + 127) / 128) {
    const int NB = (N + 15) / 16, C4 = (C + 3) / 4;
    b1 = min(b1, NB - 1);
    p0 = (const uint4*)m.w + (e * NB + b0) * C * 64 + l;
    p1 = (const uint4*)m.w + (e * NB + b1) * C * 64 + l;
    x0 = (const uint32_t*)m.exps + (e * NB + b0) * C4 * 64 + l;
    x1 = (const uint32_t*)m.exps + (e * NB + b1) * C4 * 64 + l;
  }
  struct Frag {
    uint4 a[2][2];
    uint32_t e[2];
  };
  __device__ __forceinline__ void load(Frag& f, int u) const {
    f.e[0] = x0[(u >> 1) * 64];
    f.e[1] = x1[(u >> 1) * 64];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      f.a[0][c] = f.a[1][c] = make_uint4(0u, 0u, 0u, 0u);
      if (2 * u + c < C) {
        f.a[0][c] = load_stream(p0 + (2 * u + c) * 64);
        f.a[1][c] = load_stream(p1 + (2 * u + c) * 64);
      }
    }
  }
  static constexpr int kSteps = 8;
  static __device__ __forceinline__ int at(int s, int q) { return 256 * (s >> 2) + 64 * q + 16 * (s & 3); }
  __device__ __forceinline__ bf16x8_t frag(const Frag& f, int b, int s, int u) const {
    const uint4 v = f.a[b][s >> 2];
    const uint32_t d[4] = {v.x, v.y, v.z, v.w};
    return fp4_frag(d[s & 3], fp4_scale(f.e[b], (2 * u + (s >> 2)) & 3));
  }
};

// cnt token rows times the workgroup's row pairs.  src(i): token row i (K columns);
// emit(r, i, quad, v0, v1): rows 4 quad .. + 3 of the two blocks of pair r, token
// row i.  Rows go cap (at most 16 NT) at a time; their columns through LDS in
// pieces of as many as fit.  Every wave runs every barrier; `live` says whether
// the wave's pair exists.
template <int WT, int NT, class Src, class Emit>
__device__ __forceinline__ void stream_rows(const Pair<WT>& pair, bool live, int K, int cnt, int cap, int log_ks,
                                            char* smem, int smem_bytes, int first, int step, Src src, Emit emit) {
  constexpr int U = kUnit<WT>;
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const int KS = 1 << log_ks, ks = w & (KS - 1);
  const int n = l & 15, q = l >> 4;
  const int Kpad = (K + 127) & ~127;
  for (int n0 = first; n0 < cnt; n0 += step) {
    const int rows = min(cnt - n0, cap);
    const int nt = (rows + 15) >> 4;
    const int round = U << log_ks;
    const int P = min((smem_bytes / rows - 16) / 2 / round, (K + round - 1) / round) * round;
    floatx4_t acc[2][NT];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[b][t] = floatx4_t{0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < K; p0 += P) {
      const int cols = min(P, Kpad - p0), end = min(p0 + P, K);
      const int stride = cols * 2 + 16;
      int u = p0 / U + ks;
      typename Pair<WT>::Frag cur, nxt;
      if (live && u * U < end) pair.load(cur, u);
      // token rows of this piece
      const int pc = cols >> 3;
      for (int i = tid; i < rows * pc; i += kThreads) {
        const int r = i / pc, c = i - r * pc, k = p0 + 8 * c;
        const uint4 v = k < K ? *(const uint4*)(src(n0 + r) + k) : make_uint4(0u, 0u, 0u, 0u);
        *(uint4*)(smem + r * stride + 16 * c) = v;
      }
      __syncthreads();
      if (live) {
        int row[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) row[t] = min(16 * t + n, rows - 1) * stride;
        for (; u * U < end; u += KS) {
          if ((u + KS) * U < end) pair.load(nxt, u + KS);
          const char* at = smem + (u * U - p0) * 2;
#pragma unroll
          for (int s = 0; s < Pair<WT>::kSteps; ++s) {
            if (u * U + 128 * (s >> 2) >= K) break;
            const bf16x8_t a0 = pair.frag(cur, 0, s, u), a1 = pair.frag(cur, 1, s, u);
#pragma unroll
            for (int t = 0; t < NT; ++t)
              if (t < nt) {
                const bf16x8_t bx = *(const bf16x8_t*)(at + row[t] + Pair<WT>::at(s, q));
                acc[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, bx, acc[0][t], 0, 0, 0);
                acc[1][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, bx, acc[1][t], 0, 0, 0);
              }
          }
          cur = nxt;
        }
      }
      __syncthreads();
    }
    if (log_ks == 0) {
      if (live) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (16 * t + n < rows) emit(w, n0 + 16 * t + n, q, acc[0][t], acc[1][t]);
      }
      continue;
    }
    // the KS partial sums of a pair, in order
    floatx4_t* red = (floatx4_t*)smem;
    if (live) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (16 * t + n < rows) {
          red[((w * 2 + 0) * rows + 16 * t + n) * 4 + q] = acc[0][t];
          red[((w * 2 + 1) * rows + 16 * t + n) * 4 + q] = acc[1][t];
        }
    }
    __syncthreads();
    const int per = rows * 4, total = (kWaves >> log_ks) * per;
    for (int i = tid; i < total; i += kThreads) {
      const int r = i / per, at = i - r * per;
      const floatx4_t* p = red + (r << log_ks) * 2 * per + at;
      floatx4_t v0 = p[0], v1 = p[per];
      for (int j = 1; j < KS; ++j) v0 += p[2 * j * per], v1 += p[2 * j * per + per];
      emit(r, n0 + (at >> 2), at & 3, v0, v1);
    }
    __syncthreads();
  }
}

// 16 bytes that workgroups on other XCDs read in the same launch: written through
// to memory and read past this XCD's L2 (agent-scope accesses), so that neither
// side has to write back or drop its caches.  A release fence in their place
// (every workgroup writes its XCD's L2 back) cost 32 tokens of 128 experts 39 of 128 us.
__device__ __forceinline__ void store_agent(float* p, const floatx4_t& v) {
  uint64_t* q = (uint64_t*)p;
  const uint64_t* b = (const uint64_t*)&v;
  __hip_atomic_store(q, b[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(q + 1, b[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ floatx4_t load_agent(const float* p) {
  uint64_t b[2];
  b[0] = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  b[1] = __hip_atomic_load((const uint64_t*)p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return *(const floatx4_t*)b;
}

struct DecodeArgs {
  int T, D, H, E, K, Hs;
  const bf16_t* x;      // [T, D]
  const void* idx;      // [T K]
  int is64, before;
  const float* scores;  // [T K]
  float limit;          // NaN: none
  Weights w13, w2, s13, s2;
  const float* gate;    // [T] or null: factor of the shared expert
  bf16_t* a;            // [T K, H], then [T, Hs]
  float* y;             // [T K (+ T), D]
  int* count;           // arrivals per run of output rows
  int ncount;
  bf16_t* out;          // [T, D]
  int log_ks, cap, smem_rows;
};

// The labels of the call, and which experts they hit.
struct Labels {
  short lab[kMaxSlots];   // -1: none
  short slots[kMaxSlots];  // of this workgroup's expert
  int first[kMaxE];
};

__device__ __forceinline__ void load_labels(const DecodeArgs& a, Labels& s) {
  const int S = a.T * a.K;
  for (int i = threadIdx.x; i < S; i += kThreads) {
    const int64_t v = a.is64 ? ((const int64_t*)a.idx)[i] : (int64_t)((const int*)a.idx)[i];
    const bool in = v >= 0 && v < a.E;
    s.lab[i] = in ? (short)v : (short)-1;
    if (in) s.first[v] = S;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < S; i += kThreads)
    if (s.lab[i] >= 0) atomicMin(&s.first[s.lab[i]], i);
  __syncthreads();
}

// The j-th distinct expert by its first slot (-1: fewer than that) and the number
// of distinct ones; the same in every wave.
__device__ __forceinline__ int pick_expert(const Labels& s, int S, int j, int& hit) {
  const int l = lane_id();
  int e = -1;
  hit = 0;
  for (int i0 = 0; i0 < S; i0 += 64) {
    const int i = i0 + l, lab = i < S ? s.lab[i] : -1;
    const bool lead = lab >= 0 && s.first[max(lab, 0)] == i;
    const uint64_t m = ballot64(lead);
    const uint64_t me = ballot64(lead && hit + __popcll(m & lanemask_lt()) == j);
    if (me) e = s.lab[i0 + __ffsll((unsigned long long)me) - 1];
    hit += __popcll(m);
  }
  return __builtin_amdgcn_readfirstlane(e);
}

// The slots of expert e, in order, into s.slots (every wave writes the same).
__device__ __forceinline__ int find_slots(Labels& s, int S, int e) {
  const int l = lane_id();
  int n = 0;
  for (int i0 = 0; i0 < S; i0 += 64) {
    const int i = i0 + l;
    const bool me = i < S && s.lab[i] == e;
    const uint64_t m = ballot64(me);
    if (me) s.slots[n + __popcll(m & lanemask_lt())] = (short)i;
    n += __popcll(m);
  }
  lds_wait();
  return n;
}

// out[t, d0 .. d0 + width) = the token's rows in k order, then the shared expert's.
// valid[t]: the choices of token t that name an expert.  Eight rows' loads at a time:
// one after the other, each waited for, they took 8 us of a call with one token.
__device__ __forceinline__ void sum_rows(const DecodeArgs& a, const uint32_t* valid, int d0, int width, bool shared) {
  const int S = a.T * a.K, quads = min(width, a.D - d0) / 4;
  for (int i = threadIdx.x; i < a.T * quads; i += kThreads) {
    const int t = i / quads, d = d0 + 4 * (i - t * quads);
    const uint32_t ok = valid[t];
    const float* y = a.y + (int64_t)t * a.K * a.D + d;
    floatx4_t sum = {0.f, 0.f, 0.f, 0.f}, sh = {0.f, 0.f, 0.f, 0.f};
    if (shared) sh = load_agent(a.y + (int64_t)(S + t) * a.D + d);
    for (int k0 = 0; k0 < a.K; k0 += 8) {
      floatx4_t v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)  // (rows of no expert hold nothing; they are not added)
        if (k0 + k < a.K) v[k] = load_agent(y + (int64_t)(k0 + k) * a.D);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < a.K && (ok >> (k0 + k) & 1)) sum += v[k];
    }
    sum += sh;
    *(u32x2_t*)(a.out + (int64_t)t * a.D + d) = u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
  }
}

// The choices of each token that name an expert, as bits.
__device__ __forceinline__ void note_valid(const DecodeArgs& a, const short* lab, uint32_t* valid) {
  for (int t = threadIdx.x; t < a.T; t += kThreads) {
    uint32_t m = 0;
    for (int k = 0; k < a.K; ++k) m |= (lab[t * a.K + k] >= 0 ? 1u : 0u) << k;
    valid[t] = m;
  }
}

template <int WT, int NT>
__global__ __launch_bounds__(kThreads, 4) void decode_w13_kernel(const DecodeArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  Labels& s = *(Labels*)smem;
  char* const rows = smem + sizeof(Labels);
  const int S = a.T * a.K, l = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = kWaves >> a.log_ks;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.ncount; i += kThreads) a.count[i] = 0;
  const int nsh = (a.Hs / 16 + R - 1) / R, nrb = (a.H / 16 + R - 1) / R;
  const bool shared = (int)blockIdx.x < nsh;
  const int j = shared ? 0 : ((int)blockIdx.x - nsh) / nrb;
  const int rb = shared ? blockIdx.x : (int)blockIdx.x - nsh - j * nrb;
  const int H = shared ? a.Hs : a.H;
  int e = 0, cnt = a.T;
  if (!shared) {
    load_labels(a, s);
    int hit;
    e = pick_expert(s, S, j, hit);
    if (e < 0) return;
    cnt = find_slots(s, S, e);
  }
  const int g = rb * R + (w >> a.log_ks);
  const bool live = g < H / 16;
  const Pair<WT> pair(shared ? a.s13 : a.w13, e, 2 * H, a.D, live ? g : 0, live ? H / 16 + g : 0, l);
  bf16_t* const dst = a.a + (shared ? (int64_t)S * a.H : 0);
  auto src = [&](int i) { return a.x + (int64_t)(shared ? i : s.slots[i] / a.K) * a.D; };
  auto emit = [&](int r, int i, int quad, const floatx4_t& v0, const floatx4_t& v1) {
    const int group = rb * R + r;
    if (group >= H / 16) return;
    const int slot = shared ? i : s.slots[i];
    const float sc = a.before && !shared ? a.scores[slot] : 1.f;
    float o[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      float gate = v0[v] * sc, up = v1[v] * sc;
      if (a.limit == a.limit) gate = clamp_max_nan(gate, a.limit), up = clamp_nan(up, a.limit);
      o[v] = silu_f(gate) * up;
    }
    // rounded for the matrix cores, the only rounding between x and the output
    *(u32x2_t*)(dst + (int64_t)slot * H + 16 * group + 4 * quad) = u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
  };
  stream_rows<WT, NT>(pair, live, a.D, cnt, a.cap, a.log_ks, rows, a.smem_rows, 0, a.cap, src, emit);
}

template <int WT, int NT>
__global__ __launch_bounds__(kThreads, 4) void decode_w2_kernel(const DecodeArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  __shared__ int last;
  __shared__ uint32_t valid[kDecodeMaxTokens];
  Labels& s = *(Labels*)smem;
  char* const rows = smem + sizeof(Labels);
  const int S = a.T * a.K, l = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = kWaves >> a.log_ks;
  const int nrb = (a.D / 32 + R - 1) / R, nsh = a.Hs > 0 ? nrb : 0;
  const bool shared = (int)blockIdx.x < nsh;
  const int j = shared ? 0 : ((int)blockIdx.x - nsh) / nrb;
  const int rb = shared ? blockIdx.x : (int)blockIdx.x - nsh - j * nrb;
  const int H = shared ? a.Hs : a.H;
  load_labels(a, s);
  note_valid(a, s.lab, valid);
  int hit;
  int e = pick_expert(s, S, j, hit);
  const bool none = hit == 0 && nsh == 0;  // no expert at all: the rows are zeros
  if (!shared && e < 0 && !(none && j == 0)) return;
  int cnt = a.T;
  if (shared) e = 0;
  else if (e >= 0) cnt = find_slots(s, S, e);
  if (!none) {
    const int g = rb * R + (w >> a.log_ks);
    const bool live = g < a.D / 32;
    const Pair<WT> pair(shared ? a.s2 : a.w2, e, a.D, H, live ? 2 * g : 0, live ? 2 * g + 1 : 0, l);
    const bf16_t* const from = a.a + (shared ? (int64_t)S * a.H : 0);
    auto src = [&](int i) { return from + (int64_t)(shared ? i : s.slots[i]) * H; };
    auto emit = [&](int r, int i, int quad, const floatx4_t& v0, const floatx4_t& v1) {
      const int group = rb * R + r;
      if (group >= a.D / 32) return;
      const int slot = shared ? S + i : s.slots[i];
      const float sc = shared ? (a.gate ? a.gate[i] : 1.f) : a.before ? 1.f : a.scores[slot];
      float* p = a.y + (int64_t)slot * a.D + 32 * group + 4 * quad;
      store_agent(p, v0 * sc);
      store_agent(p + 16, v1 * sc);
    };
    stream_rows<WT, NT>(pair, live, H, cnt, a.cap, a.log_ks, rows, a.smem_rows, 0, a.cap, src, emit);
    // Arrival: the workgroup's sums are in memory before it is counted, and the
    // last one reads them after its count.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
      last = __hip_atomic_fetch_add(a.count + rb, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == hit + (nsh > 0) - 1;
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(last) == 0) return;
  }
  __syncthreads();
  sum_rows(a, valid, 32 * R * rb, 32 * R, nsh > 0);
}

// ---------------------------------------------------------------------------
// bf16 weights: every wave streams its own row pairs through a ring in LDS
// ---------------------------------------------------------------------------
// What a workgroup knows of the call's labels: the hit experts in order of their
// first slot, and the slots sorted by expert.
struct Plan {
  int hit;
  short list[kMaxE];       // the j-th hit expert
  short start[kMaxE + 1];  // its first place in `sorted`
  short sorted[kMaxSlots];
  float score[kMaxSlots];  // factor of the slot at a place
  float gate[kDecodeMaxTokens];
  uint32_t valid[kDecodeMaxTokens];
};
struct PlanScratch {
  int first[kMaxE], count[kMaxE];
  short lab[kMaxSlots], pos[kMaxSlots];
};

__device__ __forceinline__ void build_plan(const DecodeArgs& a, Plan& p, PlanScratch& t, bool scored) {
  const int S = a.T * a.K, tid = threadIdx.x;
  for (int i = tid; i < S; i += kThreads) {
    const int64_t v = a.is64 ? ((const int64_t*)a.idx)[i] : (int64_t)((const int*)a.idx)[i];
    const bool in = v >= 0 && v < a.E;
    t.lab[i] = in ? (short)v : (short)-1;
    if (in) t.first[v] = S, t.count[v] = 0;
  }
  __syncthreads();
  for (int i = tid; i < S; i += kThreads)
    if (t.lab[i] >= 0) {
      atomicMin(&t.first[t.lab[i]], i);
      t.pos[i] = (short)atomicAdd(&t.count[t.lab[i]], 1);  // (columns of a tile: any order gives the same sums)
    }
  __syncthreads();
  if (tid < 64) {
    int hit = 0, base = 0;
    for (int i0 = 0; i0 < S; i0 += 64) {
      const int i = i0 + tid, lab = i < S ? t.lab[i] : -1;
      const bool lead = lab >= 0 && t.first[max(lab, 0)] == i;
      const uint64_t m = ballot64(lead);
      const int n = lead ? t.count[lab] : 0, upto = wave_inclusive_scan(n);
      if (lead) {
        const int j = hit + __popcll(m & lanemask_lt());
        p.list[j] = (short)lab;
        p.start[j] = (short)(base + upto - n);
        t.count[lab] = base + upto - n;  // from here on the expert's first place
      }
      hit += __popcll(m);
      base += __shfl(upto, 63, 64);
    }
    if (tid == 0) p.hit = hit, p.start[hit] = (short)base;
  }
  __syncthreads();
  for (int i = tid; i < S; i += kThreads)
    if (t.lab[i] >= 0) {
      const int at = t.count[t.lab[i]] + t.pos[i];
      p.sorted[at] = (short)i;
      p.score[at] = scored ? a.scores[i] : 1.f;
    }
  if (a.gate && tid < a.T) p.gate[tid] = a.gate[tid];
  note_valid(a, t.lab, p.valid);
  __syncthreads();
}

// One item of a workgroup: kWaves / KS row pairs of one expert (or the shared one).
struct Item {
  uint64_t base0, base1;  // this wave's two row blocks
  int cnt;                // token rows
  int start;              // their places in Plan::sorted; -1: the shared expert, row = token
  int rb;                 // which run of row pairs
  int K;
  bool live;              // this wave's pair exists
};

constexpr int kStageCols = 64;  // a 128-byte line of every row

// Waves that share a row pair (log2): rounds of the walk times a wave's stages in
// one (a stage is 1.4 us where HBM bounds it), the meeting of KS waves as half a
// stage.  From the experts really hit, so that the last round is full: 112 experts
// of 1536 x 2048 make 2.6 rounds with whole pairs and 21.0 with eighths.
__device__ __forceinline__ int split_log(int pairs, int K) {
  const int stages = (K + kStageCols - 1) / kStageCols, slots = kWaves * gridDim.x;
  int best = 0, cost = 0x7fffffff;
  for (int k = 0; k <= 3 && (1 << k) <= stages; ++k) {
    const int rounds = ((pairs << k) + slots - 1) / slots;
    const int c = rounds * (2 * ((stages + (1 << k) - 1) >> k) + (k > 0));
    if (c < cost) best = k, cost = c;
  }
  return best;
}

// Token rows that the partial sums of KS waves meet over at a time.
template <int NB>
constexpr int kMeetRows = NB == 1 ? 8 : NB == 2 ? 4 : 16;

// The wave's stages (32 weight rows and 8 NB token rows, 64 columns) in a ring of
// NS, filled by LDS DMA: whole 128-byte lines, eight rows an instruction, the
// 16-byte chunk c of row r at c ^ cswz(r).  The DMAs run over the flattened
// sequence of all its items' stages, NS ahead, so neither an epilogue nor the next
// expert's start empties the pipe; a wave meets the others only where KS > 1.
// item(i): the i-th item; src(item, i): byte offset of its token row i from xbase.
template <int NB, int NS, class ItemOf, class Src, class Emit>
__device__ __forceinline__ void stream_items(char* ring, floatx4_t* red, int nitems, int log_ks, uint64_t xbase,
                                             ItemOf item_of, Src src, Emit emit) {
  using namespace dma;
  constexpr int OPS = 4 + NB, SB = 1024 * OPS, NT = (NB + 1) / 2, ROWS = 8 * NB;
  const int tid = threadIdx.x, l = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KS = 1 << log_ks, ks = w & (KS - 1), G = gridDim.x;
  const int n = l & 15, q = l >> 4;
  const int lr = l >> 3;
  ring += w * (NS * SB);
  const uint32_t lds0 = lds_addr(ring);

  // the issuing end
  int it = blockIdx.x, n0 = 0, s = ks;
  bool more = it < nitems;
  Item in;
  uint32_t va[4], vb[NB];
  auto rows = [&]() {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int r = 8 * b + lr;
      vb[b] = src(in, min(n0 + r, in.cnt - 1)) + (uint32_t)(((l & 7) ^ cswz(r)) * 16);
    }
  };
  auto enter = [&]() {  // item `it`, or the next with a stage for this wave
    for (;; it += G) {
      more = it < nitems;
      if (!more) return;
      in = item_of(it);
      if (in.live && in.cnt > 0 && ks * kStageCols < in.K) break;
    }
    n0 = 0, s = ks;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      va[i] = (uint32_t)((8 * (i & 1) + lr) * in.K * 2) + (uint32_t)(((l & 7) ^ cswz(8 * i + lr)) * 16);
    rows();
  };
  auto issue = [&](int slot) {
    const uint32_t at = lds0 + (uint32_t)(slot * SB);
    const uint64_t k = (uint64_t)s * (kStageCols * 2);
    // a row's last 32 columns: the upper chunks load the lower ones again
    const bool half = (s + 1) * kStageCols > in.K;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t back = half && (((l & 7) ^ cswz(8 * i + lr)) & 4) ? 64u : 0u;
      dma16(va[i] - back, (i < 2 ? in.base0 : in.base1) + k, at + i * 1024);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint32_t back = half && (((l & 7) ^ cswz(8 * b + lr)) & 4) ? 64u : 0u;
      dma16(vb[b] - back, xbase + k, at + (4 + b) * 1024);
    }
    s += KS;
    if (s * kStageCols < in.K) return;
    s = ks;
    n0 += ROWS;
    if (n0 < in.cnt) {
      rows();
    } else {
      it += G;
      enter();
    }
  };
  enter();
  int ahead = 0;
#pragma unroll
  for (int i = 0; i < NS; ++i)
    if (more) issue(i), ++ahead;

  // the consuming end
  int slot = 0;
  for (int ci = blockIdx.x; ci < nitems; ci += G) {
    const Item c = item_of(ci);
    for (int c0 = 0; c0 < c.cnt; c0 += ROWS) {
      const int rows_here = min(c.cnt - c0, ROWS);
      floatx4_t acc[2][NT];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[b][t] = floatx4_t{0.f, 0.f, 0.f, 0.f};
      if (c.live)
        for (int cs = ks; cs * kStageCols < c.K; cs += KS) {
          if (ahead == NS) wait_vm<(NS - 1) * OPS>();
          else wait_vm<0>();
          const char* st = ring + slot * SB;
          bf16x8_t a0[2], a1[2], bx[2][NT];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int ch = 4 * h + q;
            a0[h] = *(const bf16x8_t*)(st + n * 128 + ((ch ^ cswz(n)) << 4));
            a1[h] = *(const bf16x8_t*)(st + (16 + n) * 128 + ((ch ^ cswz(16 + n)) << 4));
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const int r = (16 * t + n) & (ROWS - 1);
              bx[h][t] = *(const bf16x8_t*)(st + 4096 + r * 128 + ((ch ^ cswz(r)) << 4));
            }
          }
          lds_wait();  // the slot is free
          if (more) issue(slot);
          else --ahead;
          slot = slot == NS - 1 ? 0 : slot + 1;
          const bool half = (cs + 1) * kStageCols > c.K;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && half) break;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              acc[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0[h], bx[h][t], acc[0][t], 0, 0, 0);
              acc[1][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1[h], bx[h][t], acc[1][t], 0, 0, 0);
            }
          }
        }
      if (log_ks == 0) {
        if (c.live) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
            if (16 * t + n < rows_here) emit(c, w, c0 + 16 * t + n, q, acc[0][t], acc[1][t]);
        }
        continue;
      }
      // the KS partial sums of a pair, in order
      constexpr int MR = kMeetRows<NB>;
      for (int m0 = 0; m0 < rows_here; m0 += MR) {
        const int mr = min(rows_here - m0, MR), per = mr * 4, total = (kWaves >> log_ks) * per;
        if (c.live) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const int i = 16 * t + n - m0;
            if (i >= 0 && i < mr) {
              red[(w * 2 + 0) * per + i * 4 + q] = acc[0][t];
              red[(w * 2 + 1) * per + i * 4 + q] = acc[1][t];
            }
          }
        }
        lds_barrier();
        for (int i = tid; i < total; i += kThreads) {
          const int r = i / per, at = i - r * per;
          const floatx4_t* p = red + (r << log_ks) * 2 * per + at;
          floatx4_t v0 = p[0], v1 = p[per];
          for (int j = 1; j < KS; ++j) v0 += p[2 * j * per], v1 += p[2 * j * per + per];
          emit(c, r, c0 + m0 + (at >> 2), at & 3, v0, v1);
        }
        lds_barrier();
      }
    }
  }
  wait_vm<0>();
}

template <int NB, int NS>
constexpr int ring_bytes() {
  return kWaves * NS * 1024 * (4 + NB);
}
constexpr int kPlanBytes = (sizeof(Plan) + 1023) & ~1023;

template <int NB, int NS>
__global__ __launch_bounds__(kThreads, 2) void decode_w13_bf16_kernel(const DecodeArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  Plan& p = *(Plan*)smem;
  char* const ring = smem + kPlanBytes;
  const int S = a.T * a.K;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.ncount; i += kThreads) a.count[i] = 0;
  build_plan(a, p, *(PlanScratch*)ring, a.before != 0);
  const int hit = __builtin_amdgcn_readfirstlane(p.hit);
  const int log_ks = split_log(hit * (a.H / 16) + a.Hs / 16, a.D);
  const int R = kWaves >> log_ks, r0 = w >> log_ks;
  const int nsh = (a.Hs / 16 + R - 1) / R, nrb = (a.H / 16 + R - 1) / R;
  const int nitems = nsh + hit * nrb;
  auto item_of = [&](int i) {
    Item c;
    const bool shared = i < nsh;
    const int j = shared ? 0 : (i - nsh) / nrb;
    const int e = shared ? 0 : __builtin_amdgcn_readfirstlane(p.list[j]);
    const int H = shared ? a.Hs : a.H;
    c.rb = shared ? i : i - nsh - j * nrb;
    c.start = shared ? -1 : __builtin_amdgcn_readfirstlane(p.start[j]);
    c.cnt = shared ? a.T : __builtin_amdgcn_readfirstlane(p.start[j + 1]) - c.start;
    c.K = a.D;
    const int g = c.rb * R + r0;
    c.live = g < H / 16;
    c.base0 = (uint64_t)((const bf16_t*)(shared ? a.s13 : a.w13).w + ((int64_t)e * 2 * H + 16 * g) * a.D);
    c.base1 = c.base0 + (uint64_t)H * a.D * 2;
    return c;
  };
  auto src = [&](const Item& c, int i) {
    return (uint32_t)(c.start < 0 ? i : p.sorted[c.start + i] / a.K) * (uint32_t)a.D * 2u;
  };
  auto emit = [&](const Item& c, int r, int i, int quad, const floatx4_t& v0, const floatx4_t& v1) {
    const bool shared = c.start < 0;
    const int H = shared ? a.Hs : a.H, group = c.rb * R + r;
    if (group >= H / 16) return;
    const int slot = shared ? i : p.sorted[c.start + i];
    const float sc = shared ? 1.f : p.score[c.start + i];
    bf16_t* const dst = a.a + (shared ? (int64_t)S * a.H : 0) + (int64_t)slot * H + 16 * group + 4 * quad;
    float o[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      float gate = v0[v] * sc, up = v1[v] * sc;
      if (a.limit == a.limit) gate = clamp_max_nan(gate, a.limit), up = clamp_nan(up, a.limit);
      o[v] = silu_f(gate) * up;
    }
    // rounded for the matrix cores, the only rounding between x and the output
    *(u32x2_t*)dst = u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
  };
  stream_items<NB, NS>(ring, (floatx4_t*)(ring + ring_bytes<NB, NS>()), nitems, log_ks, (uint64_t)a.x, item_of, src,
                       emit);
}

template <int NB, int NS>
__global__ __launch_bounds__(kThreads, 2) void decode_w2_bf16_kernel(const DecodeArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  __shared__ int nlast;
  Plan& p = *(Plan*)smem;
  char* const ring = smem + kPlanBytes;
  const int S = a.T * a.K;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  build_plan(a, p, *(PlanScratch*)ring, a.before == 0);
  const int hit = __builtin_amdgcn_readfirstlane(p.hit);
  const int log_ks = split_log((hit + (a.Hs > 0)) * (a.D / 32), hit > 0 ? a.H : a.Hs);
  const int R = kWaves >> log_ks, r0 = w >> log_ks;
  const int nrb = (a.D / 32 + R - 1) / R, nsh = a.Hs > 0 ? nrb : 0;
  const int nitems = nsh + hit * nrb;
  auto item_of = [&](int i) {
    Item c;
    const bool shared = i < nsh;
    const int j = shared ? 0 : (i - nsh) / nrb;
    const int e = shared ? 0 : __builtin_amdgcn_readfirstlane(p.list[j]);
    c.rb = shared ? i : i - nsh - j * nrb;
    c.start = shared ? -1 : __builtin_amdgcn_readfirstlane(p.start[j]);
    c.cnt = shared ? a.T : __builtin_amdgcn_readfirstlane(p.start[j + 1]) - c.start;
    c.K = shared ? a.Hs : a.H;
    const int g = c.rb * R + r0;
    c.live = g < a.D / 32;
    c.base0 = (uint64_t)((const bf16_t*)(shared ? a.s2 : a.w2).w + ((int64_t)e * a.D + 32 * g) * c.K);
    c.base1 = c.base0 + (uint64_t)c.K * 32;
    return c;
  };
  const uint32_t shared_at = (uint32_t)S * (uint32_t)a.H * 2u;
  auto src = [&](const Item& c, int i) {
    return c.start < 0 ? shared_at + (uint32_t)i * (uint32_t)a.Hs * 2u
                       : (uint32_t)p.sorted[c.start + i] * (uint32_t)a.H * 2u;
  };
  auto emit = [&](const Item& c, int r, int i, int quad, const floatx4_t& v0, const floatx4_t& v1) {
    const int group = c.rb * R + r;
    if (group >= a.D / 32) return;
    const bool shared = c.start < 0;
    const int slot = shared ? S + i : p.sorted[c.start + i];
    const float sc = shared ? (a.gate ? p.gate[i] : 1.f) : p.score[c.start + i];
    float* y = a.y + (int64_t)slot * a.D + 32 * group + 4 * quad;
    store_agent(y, v0 * sc);
    store_agent(y + 16, v1 * sc);
  };
  if (threadIdx.x == 0) nlast = 0;
  stream_items<NB, NS>(ring, (floatx4_t*)(ring + ring_bytes<NB, NS>()), nitems, log_ks, (uint64_t)a.a, item_of, src,
                       emit);
  // Arrivals: the workgroup's sums are in memory (the stream ends waiting for its
  // stores) before its items are counted; who brings a run of rows to its count
  // reads the others' sums after that.
  __syncthreads();
  short* const last = (short*)ring;
  const int all = hit + (nsh > 0);
  if (all > 0) {
    for (int i = threadIdx.x; i * (int)gridDim.x + (int)blockIdx.x < nitems; i += kThreads) {
      const int it = i * gridDim.x + blockIdx.x, rb = it < nsh ? it : (it - nsh) % nrb;
      if (__hip_atomic_fetch_add(a.count + rb, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1)
        last[atomicAdd(&nlast, 1)] = (short)rb;
    }
  } else {  // no expert at all: the rows are zeros
    for (int rb = blockIdx.x + threadIdx.x * gridDim.x; rb < nrb; rb += kThreads * gridDim.x)
      last[atomicAdd(&nlast, 1)] = (short)rb;
  }
  __syncthreads();
  for (int f = 0; f < nlast; ++f) sum_rows(a, p.valid, 32 * R * last[f], 32 * R, nsh > 0);
}

// z[t, e] = bf16(sum_d x[t, d] w[e, d]).  Products of bf16 pairs are exact in 64
// bits and so are nearly all their sums, so a logit does not depend on the order
// of its terms and equal inputs give equal picks in every batch.  Row E: the
// shared expert's gate, through a sigmoid.  A wave takes one row and TB tokens,
// eight columns per lane and step, kAhead steps' loads at a time.
constexpr int kAhead = 4;
template <int TB>
__global__ __launch_bounds__(256) void router_logits_kernel(const bf16_t* __restrict__ x,
                                                            const bf16_t* __restrict__ w_router,
                                                            const bf16_t* __restrict__ w_gate, int T, int E, int D,
                                                            bf16_t* __restrict__ logits, float* __restrict__ gate) {
  const int l = threadIdx.x & 63;
  const int e = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = blockIdx.y * TB;
  if (e >= E + (w_gate != nullptr)) return;
  const bf16_t* w = e < E ? w_router + (int64_t)e * D : w_gate;
  double acc[TB];
#pragma unroll
  for (int t = 0; t < TB; ++t) acc[t] = 0.0;
  for (int k0 = 8 * l; k0 < D; k0 += 512 * kAhead) {
    uint4 wv[kAhead], xv[kAhead][TB];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k = min(k0 + 512 * j, D - 8);
      wv[j] = *(const uint4*)(w + k);
#pragma unroll
      for (int t = 0; t < TB; ++t) xv[j][t] = *(const uint4*)(x + (int64_t)min(t0 + t, T - 1) * D + k);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (k0 + 512 * j >= D) break;
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
    if (l == t && t0 + t < T) {
      const uint32_t z = f32_to_bf16((float)v);
      if (e < E) logits[(int64_t)(t0 + t) * E + e] = (bf16_t)z;
      else gate[t0 + t] = 1.f / (1.f + expf(-bf16_to_f32(z)));
    }
  }
}

// out[m] = x[m] w[e]^T (+ bias) in bf16; expert e's rows offs[e - 1] .. offs[e] - 1,
// or all of them without offs.
struct Fp4Args {
  const bf16_t* x;
  Weights w;
  const int* offs;
  const void* bias;
  int bias32, M, E, N, K;
  bf16_t* out;
  int log_ks, cap, smem_rows;
};

template <int NT>
__global__ __launch_bounds__(kThreads, 4) void grouped_mm_fp4_kernel(const Fp4Args a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int l = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int R = kWaves >> a.log_ks;
  const int NB = (a.N + 15) / 16, NP = (NB + 1) / 2, nrb = (NP + R - 1) / R;
  const int e = blockIdx.x / nrb, rb = blockIdx.x - e * nrb;
  int r0 = 0, r1 = a.M;
  if (a.offs) {
    r0 = e > 0 ? min(max(a.offs[e - 1], 0), a.M) : 0;
    r1 = min(max(a.offs[e], 0), a.M);
  }
  const int cnt = r1 - r0, first = (int)blockIdx.y * a.cap;
  if (first >= cnt) return;
  const int g = rb * R + (w >> a.log_ks);
  const bool live = g < NP;
  const Pair<W_FP4> pair(a.w, e, a.N, a.K, live ? 2 * g : 0, live ? 2 * g + 1 : 0, l);
  auto src = [&](int i) { return a.x + (int64_t)(r0 + i) * a.K; };
  auto emit = [&](int r, int i, int quad, const floatx4_t& v0, const floatx4_t& v1) {
    const int group = rb * R + r;
    if (group >= NP) return;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int n = 32 * group + 16 * b + 4 * quad;
      floatx4_t v = b ? v1 : v0;
      bf16_t* p = a.out + (int64_t)(r0 + i) * a.N + n;
      if (a.bias)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (n + c < a.N) v[c] += a.bias32 ? ((const float*)a.bias)[n + c] : bf16_to_f32(((const bf16_t*)a.bias)[n + c]);
      if ((a.N & 3) == 0) {
        if (n < a.N) *(u32x2_t*)p = u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (n + c < a.N) p[c] = (bf16_t)f32_to_bf16(v[c]);
      }
    }
  };
  stream_rows<W_FP4, NT>(pair, live, a.K, cnt, a.cap, a.log_ks, smem, a.smem_rows, first, a.cap * gridDim.y, src, emit);
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Waves that share a row pair (log2): as many as bring the launch to two
// workgroups per CU, while each keeps a unit of columns and, with 64 token rows at
// a time, a piece of KS units fits the LDS.
int pick_log_ks(int64_t pairs, int K, int unit, int cap) {
  int log_ks = 0;
  while (log_ks < 3 && pairs * (1 << log_ks) / kWaves < 2 * num_cus() && (unit << (log_ks + 1)) <= K &&
         (int64_t)cap * ((unit << (log_ks + 1)) * 2 + 16) <= kRowBytes)
    ++log_ks;
  return log_ks;
}

// LDS for the rows of a pass: all their columns if they fit; the partial sums of
// KS waves need 2 KB for each 16 rows and wave.
int row_bytes(int cap, int K, int log_ks, int unit) {
  const int kpad = (K + (unit << log_ks) - 1) / (unit << log_ks) * (unit << log_ks);
  const int64_t all = (int64_t)cap * (kpad * 2 + 16), red = log_ks > 0 ? (int64_t)cap * kWaves * 128 : 0;
  return (int)std::min<int64_t>(kRowBytes, std::max(all, red));
}

hipError_t launch_experts_fp4(DecodeArgs a, hipStream_t stream) {
  constexpr int WT = W_FP4, U = kUnit<WT>;
  const int S = a.T * a.K, hit = std::min(a.E, S);
  const bool few = a.T <= 16;
  a.cap = few ? a.T : std::min(a.T, 64);
  // (first launch) gate and up rows of 16 hidden units to a pair
  a.log_ks = pick_log_ks((int64_t)hit * (a.H / 16) + a.Hs / 16, a.D, U, a.cap);
  a.smem_rows = row_bytes(a.cap, a.D, a.log_ks, U);
  int R = kWaves >> a.log_ks;
  const int log_ks2 = pick_log_ks((int64_t)(hit + (a.Hs > 0)) * (a.D / 32), std::max(a.H, a.Hs), U, a.cap);
  const int R2 = kWaves >> log_ks2, nrb2 = ceil_div(a.D / 32, R2);
  a.ncount = nrb2;
  dim3 grid(ceil_div(a.Hs / 16, R) + hit * ceil_div(a.H / 16, R));
  auto k13 = few ? decode_w13_kernel<WT, 1> : decode_w13_kernel<WT, 4>;
  const uint32_t lds13 = sizeof(Labels) + a.smem_rows;
  hipError_t err = hipFuncSetAttribute((const void*)k13, hipFuncAttributeMaxDynamicSharedMemorySize, lds13);
  if (err != hipSuccess) return err;
  err = launch_k(false, k13, grid, dim3(kThreads), lds13, stream, a);
  if (err != hipSuccess) return err;
  a.log_ks = log_ks2;
  a.smem_rows = row_bytes(a.cap, std::max(a.H, a.Hs), log_ks2, U);
  grid = dim3(((a.Hs > 0) + hit) * nrb2);
  auto k2 = few ? decode_w2_kernel<WT, 1> : decode_w2_kernel<WT, 4>;
  const uint32_t lds2 = sizeof(Labels) + a.smem_rows;
  err = hipFuncSetAttribute((const void*)k2, hipFuncAttributeMaxDynamicSharedMemorySize, lds2);
  if (err != hipSuccess) return err;
  return launch_k(false, k2, grid, dim3(kThreads), lds2, stream, a);
}

template <int NB, int NS>
hipError_t launch_bf16(DecodeArgs a, hipStream_t stream) {
  constexpr uint32_t lds = kPlanBytes + ring_bytes<NB, NS>() + kMeetRows<NB> * kWaves * 128;
  static_assert(lds + 1024 <= 160 * 1024, "LDS");
  const int hit = std::min(a.E, a.T * a.K), G = num_cus();
  a.ncount = a.D / 32;
  auto k13 = decode_w13_bf16_kernel<NB, NS>;
  auto k2 = decode_w2_bf16_kernel<NB, NS>;
  // (one item per row pair at the finest)
  hipError_t err = hipFuncSetAttribute((const void*)k13, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (err != hipSuccess) return err;
  err = launch_k(false, k13, dim3(std::min<int64_t>((int64_t)hit * (a.H / 16) + a.Hs / 16, G)), dim3(kThreads), lds, stream, a);
  if (err != hipSuccess) return err;
  err = hipFuncSetAttribute((const void*)k2, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (err != hipSuccess) return err;
  return launch_k(false, k2, dim3(std::min<int64_t>((int64_t)(hit + (a.Hs > 0)) * (a.D / 32), G)), dim3(kThreads), lds, stream, a);
}

// Token rows per pass, by the rows that an expert gets on average: a pass more
// streams its weights again, a larger one takes LDS from the ring.
hipError_t launch_experts_bf16(const DecodeArgs& a, hipStream_t stream) {
  const int most = a.Hs > 0 ? a.T : 0, rows = std::max(most, ceil_div(a.T * a.K, a.E));
  if (a.T <= 8 || rows <= 4) return launch_bf16<1, 3>(a, stream);
  return rows <= 10 ? launch_bf16<2, 3>(a, stream) : launch_bf16<4, 2>(a, stream);
}

size_t al256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

size_t router_decode_workspace_bytes(int64_t T, int E) { return al256((size_t)T * E * 2); }

hipError_t launch_router_decode(const void* x, const void* w_router, const void* w_gate, const float* bias, int T, int E,
                                int D, int K, const RouterGroups& groups, int score_func, int renorm, float renorm_eps,
                                float route_scale, float* top_scores, int64_t* top_idx, float* gate, void* logits,
                                hipStream_t stream) {
  const int rows = E + (w_gate != nullptr);
  const int tb = T >= 4 ? 4 : T >= 2 ? 2 : 1;
  const dim3 grid(ceil_div(rows, 4), ceil_div(T, tb));
  auto kernel = tb == 4 ? router_logits_kernel<4> : tb == 2 ? router_logits_kernel<2> : router_logits_kernel<1>;
  hipError_t err = launch_k(false, kernel, grid, dim3(256), 0, stream, (const bf16_t*)x, (const bf16_t*)w_router,
                            (const bf16_t*)w_gate, T, E, D, (bf16_t*)logits, gate);
  if (err != hipSuccess) return err;
  return launch_router_topk_grouped(logits, true, bias, T, E, K, groups, score_func, renorm, renorm_eps, route_scale,
                                    top_scores, top_idx, stream);
}

// Workspace: activations of the slots and of the shared expert, their fp32 output
// rows, arrival counters.
size_t experts_decode_workspace_bytes(int64_t T, int64_t D, int64_t H, int K, int64_t Hs) {
  const int64_t S = T * K;
  return al256((size_t)(S * H + (Hs > 0 ? T * Hs : 0)) * 2) + al256((size_t)(S + (Hs > 0 ? T : 0)) * D * 4) +
         al256((size_t)(D / 32) * 4);
}

hipError_t launch_experts_decode(const ExpertsDecode& c, void* ws, hipStream_t stream) {
  DecodeArgs a{};
  a.T = c.T, a.D = c.D, a.H = c.H, a.E = c.E, a.K = c.K, a.Hs = c.Hs;
  a.x = (const bf16_t*)c.x;
  a.idx = c.idx, a.is64 = c.is64, a.before = c.before;
  a.scores = c.scores, a.limit = c.limit, a.gate = c.gate;
  a.w13 = {c.w13, c.e13}, a.w2 = {c.w2, c.e2}, a.s13 = {c.s13, c.es13}, a.s2 = {c.s2, c.es2};
  const int64_t S = (int64_t)a.T * a.K, Ts = a.Hs > 0 ? a.T : 0;
  char* p = (char*)ws;
  a.a = (bf16_t*)p;
  p += al256((size_t)(S * a.H + Ts * a.Hs) * 2);
  a.y = (float*)p;
  p += al256((size_t)(S + Ts) * a.D * 4);
  a.count = (int*)p;
  a.out = (bf16_t*)c.out;
  return c.fp4 ? launch_experts_fp4(a, stream) : launch_experts_bf16(a, stream);
}

hipError_t launch_grouped_mm_fp4(const void* x, const void* codes, const void* exps, const int* offs, const void* bias,
                                 bool bias32, int M, int E, int N, int K, void* out, hipStream_t stream) {
  Fp4Args a{};
  a.x = (const bf16_t*)x, a.w = {codes, (const uint8_t*)exps}, a.offs = offs, a.bias = bias, a.bias32 = bias32;
  a.M = M, a.E = E, a.N = N, a.K = K, a.out = (bf16_t*)out;
  const bool few = M <= 16;
  a.cap = few ? M : std::min(M, 64);
  const int pairs = ceil_div(ceil_div(N, 16), 2), tiles = std::min(ceil_div(M, a.cap), 1024);
  a.log_ks = pick_log_ks((int64_t)pairs * (offs ? std::min(E, M) : tiles), K, kUnit<W_FP4>, a.cap);
  a.smem_rows = row_bytes(a.cap, K, a.log_ks, kUnit<W_FP4>);
  auto kernel = few ? grouped_mm_fp4_kernel<1> : grouped_mm_fp4_kernel<4>;
  const hipError_t err =
      hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, a.smem_rows);
  if (err != hipSuccess) return err;
  const dim3 grid(E * ceil_div(pairs, kWaves >> a.log_ks), offs ? std::min(tiles, 8) : tiles);
  return launch_k(false, kernel, grid, dim3(kThreads), a.smem_rows, stream, a);
}

}  // namespace ttamd
