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
#include "router_select.h"

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
  const char* plan;
  int plan_lds;         // its bytes in LDS
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
    *(u32x2_t*)(dst + (int64_t)slot * H + 16 * group + 4 * quad) = activate(v0 * sc, v1 * sc, a.limit);
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
// The plan: which experts are hit, and by which slots
// ---------------------------------------------------------------------------
// One workgroup makes it (with the selection, where the router runs), the two
// streaming kernels copy it to LDS.  Hit experts in order; slots sorted by expert
// ("places").
struct PlanMap {
  int T, S;
  __host__ __device__ constexpr int valid() const { return 16; }                   // uint32 [T]: choices that name an expert
  __host__ __device__ constexpr int gate() const { return valid() + 4 * T; }       // float [T]: factor of the shared expert
  __host__ __device__ constexpr int score() const { return gate() + 4 * T; }       // float [S], by place
  __host__ __device__ constexpr int sorted() const { return score() + 4 * S; }     // short [S]: slot at a place
  __host__ __device__ constexpr int inverse() const { return sorted() + 2 * S; }   // short [S]: place of a slot
  __host__ __device__ constexpr int list() const { return inverse() + 2 * S; }     // short [hit]: experts
  __host__ __device__ constexpr int start() const { return list() + 2 * S; }       // short [hit + 1]: their first places
  __host__ __device__ constexpr int bytes() const { return (start() + 2 * (S + 1) + 15) & ~15; }  // int hit at 0
};
constexpr int kMaxPlanBytes = PlanMap{kDecodeMaxTokens, kMaxSlots}.bytes();

struct Plan : PlanMap {
  char* p;
  __device__ Plan(char* p_, int T_, int S_) : PlanMap{T_, S_}, p(p_) {}
  __device__ int& hit() const { return *(int*)p; }
  __device__ uint32_t& valid(int i) const { return ((uint32_t*)(p + PlanMap::valid()))[i]; }
  __device__ float& gate(int i) const { return ((float*)(p + PlanMap::gate()))[i]; }
  __device__ float& score(int i) const { return ((float*)(p + PlanMap::score()))[i]; }
  __device__ short& sorted(int i) const { return ((short*)(p + PlanMap::sorted()))[i]; }
  __device__ short& inverse(int i) const { return ((short*)(p + PlanMap::inverse()))[i]; }
  __device__ short& list(int i) const { return ((short*)(p + PlanMap::list()))[i]; }
  __device__ short& start(int i) const { return ((short*)(p + PlanMap::start()))[i]; }
};

constexpr int kPlanThreads = 1024;

struct PlanArgs {
  select::GroupTopkArgs topk;  // of the selection (its scores and idx are outputs)
  const void* idx;             // without it: given picks
  int is64;
  const float* scores;
  const float* gate;           // [T] or null: 1
  int T, E, K;
  char* plan;
  int* count;                  // cleared for the kernels after this one
  int ncount;
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
  for (int i = tid; i < a.ncount; i += kPlanThreads) a.count[i] = 0;
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
  if (tid == 0) p.hit() = hits;
  dma::lds_barrier();
  if (mine >= 0) {
    const int at = total[mine] + pos;
    p.sorted(at) = (short)tid;
    p.inverse(tid) = (short)at;
    p.score(at) = score[tid];
  }
}

// ---------------------------------------------------------------------------
// Streams: every wave pulls its own weight rows through a ring in LDS
// ---------------------------------------------------------------------------
// A stage of a wave: its weight rows and the token rows over kCols columns (bf16: a
// 128-byte line of every row; 4 bits: one tile and its exponents).  A DMA
// instruction moves 8 bf16 weight rows, one 4-bit tile of 16, or 8 (4) token rows of
// 128 (256) bytes; BL and NB count the instructions.
template <int WT, int BL, int NB, int NS>
struct Ring {
  static constexpr int kCols = WT == W_BF16 ? 64 : 128;
  static constexpr int kBlocks = WT == W_BF16 ? (BL + 1) / 2 : BL;  // of 16 rows
  static constexpr int kExps = BL * 1024;                           // 4 bits: 256 bytes of exponents per block
  static constexpr int kRowsAt = kExps + (WT == W_BF16 ? 0 : 256 * BL);
  static constexpr int kBytes = kRowsAt + 1024 * NB;
  static constexpr int kOps = (WT == W_BF16 ? BL : 2 * BL) + NB;
  static constexpr int kRows = NB * (WT == W_BF16 ? 8 : 4);
  static constexpr int NT = (kRows + 15) / 16;
  static constexpr int kAll = kWaves * NS * kBytes;
};

// One item of a wave: rows of one expert (or the shared one) times its token rows.
template <int BL>
struct Item {
  uint64_t base[BL];  // per load: bf16, its first row of 8; 4 bits, its first tile
  uint64_t exps[BL];  // 4 bits: its exponents
  int cnt;            // token rows
  int start;          // their first place in the plan; -1: the shared expert, row = token
  int rb;             // which run of rows (the caller's)
  int K;
  bool live;          // the wave has rows here
};

// Runs the items first, first + step, ... < nitems.  Of a item's stages the wave
// takes every KS-th from ks on.  The DMAs run over the flattened sequence of all
// its stages, NS ahead, so neither an epilogue nor the next expert's start empties
// the pipe, and no wave waits for another here.  item_of(i): the i-th item;
// src(item, i): byte offset of its token row i from xbase; done(item, c0, rows,
// acc): the sums of its token rows c0 .. c0 + rows - 1 (lane l, block b, tile t:
// weight rows 4 (l / 16) .. + 3, token row c0 + 16 t + l % 16).
template <int WT, int BL, int NB, int NS, class ItemOf, class Src, class Done>
__device__ __forceinline__ void stream_items(char* ring, int first, int step, int nitems, int ks, int KS,
                                             uint64_t xbase, ItemOf item_of, Src src, Done done) {
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

  // the issuing end
  int it = first, n0 = 0, s = ks;
  bool more = it < nitems;
  Item<BL> in;
  uint32_t va[BL], vb[NB];
  auto rows = [&]() {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int r = WT == W_BF16 ? 8 * b + (l >> 3) : 4 * b + (l >> 4);
      const int ch = WT == W_BF16 ? chunk8(b) : chunk16(b);
      vb[b] = src(in, min(n0 + r, in.cnt - 1)) + (uint32_t)(16 * ch);
    }
  };
  auto enter = [&]() {  // item `it`, or the next with a stage for this wave
    for (;; it += step) {
      more = it < nitems;
      if (!more) return;
      in = item_of(it);
      if (in.live && in.cnt > 0 && ks * R::kCols < in.K) break;
    }
    n0 = 0, s = ks;
    if constexpr (WT == W_BF16) {
#pragma unroll
      for (int i = 0; i < BL; ++i) va[i] = (uint32_t)((l >> 3) * in.K * 2) + (uint32_t)(16 * chunk8(i));
    }
    rows();
  };
  auto issue = [&](int slot) {
    const uint32_t at = lds0 + (uint32_t)(slot * R::kBytes);
    const int left = in.K - s * R::kCols;  // columns of the row from this stage on, a multiple of 32
    if constexpr (WT == W_BF16) {
      const uint64_t k = (uint64_t)s * 128;
#pragma unroll
      for (int i = 0; i < BL; ++i) {  // past the row's end: the chunk 64 bytes before once more
        const uint32_t back = left < 64 && (chunk8(i) & 4) ? 64u : 0u;
        dma16(va[i] - back, in.base[i] + k, at + i * 1024);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint32_t back = left < 64 && (chunk8(b) & 4) ? 64u : 0u;
        dma16(vb[b] - back, xbase + k, at + R::kRowsAt + b * 1024);
      }
    } else {
#pragma unroll
      for (int b = 0; b < BL; ++b) dma16((uint32_t)(16 * l), in.base[b] + (uint64_t)s * 1024, at + b * 1024);
#pragma unroll
      for (int b = 0; b < BL; ++b)
        dma4((uint32_t)(4 * l), in.exps[b] + (uint64_t)(s >> 2) * 256, at + R::kExps + b * 256);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int ch = chunk16(b);
        const uint32_t back = 8 * ch >= left ? (uint32_t)(16 * (ch & ~3)) : 0u;
        dma16(vb[b] - back, xbase + (uint64_t)s * 256, at + R::kRowsAt + b * 1024);
      }
    }
    s += KS;
    if (s * R::kCols < in.K) return;
    s = ks;
    n0 += R::kRows;
    if (n0 < in.cnt) {
      rows();
    } else {
      it += step;
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
  for (int ci = first; ci < nitems; ci += step) {
    const Item<BL> c = item_of(ci);
    for (int c0 = 0; c0 < c.cnt; c0 += R::kRows) {
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
            uint4 qw[BL];
            float scale[BL];
            bf16x8_t bx[4][NT];
#pragma unroll
            for (int b = 0; b < BL; ++b) {
              qw[b] = *(const uint4*)(st + b * 1024 + 16 * l);
              scale[b] = fp4_scale(*(const uint32_t*)(st + R::kExps + b * 256 + 4 * l), cs & 3);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                const int r = (16 * t + n) & (R::kRows - 1);
                bx[j][t] = *(const bf16x8_t*)(st + R::kRowsAt + r * 256 + (((4 * q + j) ^ (r & 15)) << 4));
              }
            lds_wait();
            if (more) issue(slot);
            else --ahead;
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
          slot = slot == NS - 1 ? 0 : slot + 1;
        }
      done(c, c0, min(c.cnt - c0, R::kRows), acc);
    }
  }
  wait_vm<0>();
}

// Waves that share an item (log2) out of kWaves: rounds of the walk times a wave's
// stages in one, twice, with `meet` for the meeting of KS waves.  From the experts
// really hit, so that the last round is full: 112 experts of 1536 x 2048 make 2.6
// rounds with whole row pairs and 21.0 with eighths.
__device__ __forceinline__ int split_log(int items, int slots, int stages, int most, int meet) {
  int best = 0, cost = 0x7fffffff;
  for (int k = 0; k <= most && (1 << k) <= stages; ++k) {
    const int rounds = ((items << k) + slots - 1) / slots;
    const int c = rounds * (2 * ((stages + (1 << k) - 1) >> k) + (k > 0 ? meet : 0));
    if (c < cost) best = k, cost = c;
  }
  return best;
}

// Load b of an item: 8 rows (bf16) or 16 (4 bits) of expert e's [N, K] weights from
// row `row` on.
template <int WT, int BL>
__device__ __forceinline__ void set_load(Item<BL>& c, int b, const Weights& m, int64_t e, int N, int K, int row) {
  if constexpr (WT == W_BF16) {
    c.base[b] = (uint64_t)((const bf16_t*)m.w + (e * N + row) * K);
  } else {
    const int C = (K + 127) / 128, C4 = (C + 3) / 4;
    const int64_t at = e * ((N + 15) / 16) + row / 16;
    c.base[b] = (uint64_t)((const char*)m.w + at * C * 1024);
    c.exps[b] = (uint64_t)(m.exps + at * C4 * 256);
  }
}

__device__ __forceinline__ void load_plan(const DecodeArgs& a, char* smem) {
  const int n = PlanMap{a.T, a.T * a.K}.bytes() / 16;
  for (int i = threadIdx.x; i < n; i += kThreads) ((uint4*)smem)[i] = ((const uint4*)a.plan)[i];
  __syncthreads();
}

// Token rows that the partial sums of KS waves meet over at a time (1 KB each).
constexpr int kMeetRows = 4;

// gate and up rows of 16 hidden units
template <int WT>
constexpr int kPairLoads = WT == W_BF16 ? 4 : 2;

template <int WT, int NB, int NS>
__global__ __launch_bounds__(kThreads, 2) void stream_w13_kernel(const DecodeArgs a) {
  constexpr int BL = kPairLoads<WT>;
  using Rg = Ring<WT, BL, NB, NS>;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int S = a.T * a.K, tid = threadIdx.x, l = tid & 63;
  const Plan p(smem, a.T, S);
  char* const ring = smem + a.plan_lds;
  floatx4_t* const red = (floatx4_t*)(ring + Rg::kAll);
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  load_plan(a, smem);
  const int hit = __builtin_amdgcn_readfirstlane(p.hit());
  const int log_ks = split_log(hit * (a.H / 16) + a.Hs / 16, kWaves * gridDim.x,
                               (a.D + Rg::kCols - 1) / Rg::kCols, 3, 1);
  const int KS = 1 << log_ks, R = kWaves >> log_ks, r0 = w >> log_ks;
  const int nsh = (a.Hs / 16 + R - 1) / R, nrb = (a.H / 16 + R - 1) / R;
  auto item_of = [&](int i) {
    Item<BL> c;
    const bool shared = i < nsh;
    const int j = shared ? 0 : (i - nsh) / nrb;
    const int e = shared ? 0 : __builtin_amdgcn_readfirstlane(p.list(j));
    const int H = shared ? a.Hs : a.H;
    c.rb = shared ? i : i - nsh - j * nrb;
    c.start = shared ? -1 : __builtin_amdgcn_readfirstlane(p.start(j));
    c.cnt = shared ? a.T : __builtin_amdgcn_readfirstlane(p.start(j + 1)) - c.start;
    c.K = a.D;
    const int g = c.rb * R + r0;
    c.live = g < H / 16;
    const Weights& m = shared ? a.s13 : a.w13;
#pragma unroll
    for (int b = 0; b < BL; ++b)
      set_load<WT>(c, b, m, e, 2 * H, a.D, (b < BL / 2 ? 0 : H) + 16 * g + (WT == W_BF16 ? 8 * (b & 1) : 0));
    return c;
  };
  auto src = [&](const Item<BL>& c, int i) {
    return (uint32_t)(c.start < 0 ? i : p.sorted(c.start + i) / a.K) * (uint32_t)a.D * 2u;
  };
  auto emit = [&](const Item<BL>& c, int r, int i, int quad, const floatx4_t& v0, const floatx4_t& v1) {
    const bool shared = c.start < 0;
    const int H = shared ? a.Hs : a.H, group = c.rb * R + r;
    if (group >= H / 16) return;
    const int slot = shared ? i : p.sorted(c.start + i);
    const float sc = shared || !a.before ? 1.f : p.score(c.start + i);
    bf16_t* const dst = a.a + (shared ? (int64_t)S * a.H : 0) + (int64_t)slot * H + 16 * group + 4 * quad;
    *(u32x2_t*)dst = activate(v0 * sc, v1 * sc, a.limit);
  };
  stream_items<WT, BL, NB, NS>(
      ring, blockIdx.x, gridDim.x, nsh + hit * nrb, w & (KS - 1), KS, (uint64_t)a.x, item_of, src,
      [&](const Item<BL>& c, int c0, int rows, const floatx4_t (&acc)[2][Rg::NT]) {
        constexpr int NT = Rg::NT;
        const int n = l & 15, q = l >> 4;
        if (log_ks == 0) {
          if (c.live) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
              if (16 * t + n < rows) emit(c, w, c0 + 16 * t + n, q, acc[0][t], acc[1][t]);
          }
          return;
        }
        // the KS partial sums of a pair, in order
        for (int m0 = 0; m0 < rows; m0 += kMeetRows) {
          const int mr = min(rows - m0, kMeetRows), per = mr * 4, total = R * per;
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
          dma::lds_barrier();
          for (int i = tid; i < total; i += kThreads) {
            const int r = i / per, at = i - r * per;
            const floatx4_t* v = red + (r << log_ks) * 2 * per + at;
            floatx4_t v0 = v[0], v1 = v[per];
            for (int j = 1; j < KS; ++j) v0 += v[2 * j * per], v1 += v[2 * j * per + per];
            emit(c, r, c0 + m0 + (at >> 2), at & 3, v0, v1);
          }
          dma::lds_barrier();
        }
      });
}

// A workgroup owns the output rows of BL loads (8 each, 4 bits: 16) for every
// expert; its waves (KS to a share of
// the columns) take the hit experts in turn, the weighted rows of all slots meet in
// LDS and leave as the tokens' sums: nothing goes through memory, no workgroup
// waits for another, every sum has its order.
template <int WT, int BL, int NB, int NS>
__global__ __launch_bounds__(kThreads, 2) void stream_w2_kernel(const DecodeArgs a) {
  using Rg = Ring<WT, BL, NB, NS>;
  constexpr int MB = Rg::kBlocks, LR = WT == W_BF16 ? 8 : 16;  // rows of a load
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int S = a.T * a.K, tid = threadIdx.x, l = tid & 63;
  const Plan p(smem, a.T, S);
  char* const ring = smem + a.plan_lds;
  floatx4_t* const sums = (floatx4_t*)(ring + Rg::kAll);  // [KS][place][MB][4]
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  load_plan(a, smem);
  const int hit = __builtin_amdgcn_readfirstlane(p.hit());
  const int nsh = a.Hs > 0, places = S + (nsh ? a.T : 0);
  constexpr int C = Rg::kCols;
  const int log_ks = split_log(hit + nsh, kWaves, ((hit > 0 ? a.H : a.Hs) + C - 1) / C, a.log_ks, 0);
  const int KS = 1 << log_ks, R = kWaves >> log_ks, ks = w & (KS - 1);
  const int row0 = blockIdx.x * BL * LR;
  auto item_of = [&](int i) {
    Item<BL> c;
    const bool shared = i < nsh;
    const int e = shared ? 0 : __builtin_amdgcn_readfirstlane(p.list(i - nsh));
    c.rb = 0;
    c.start = shared ? -1 : __builtin_amdgcn_readfirstlane(p.start(i - nsh));
    c.cnt = shared ? a.T : __builtin_amdgcn_readfirstlane(p.start(i - nsh + 1)) - c.start;
    c.K = shared ? a.Hs : a.H;
    c.live = true;
#pragma unroll
    for (int b = 0; b < BL; ++b)  // (rows past the last: the last ones again, not stored)
      set_load<WT>(c, b, shared ? a.s2 : a.w2, e, a.D, c.K, min(row0 + b * LR, a.D - LR));
    return c;
  };
  const uint32_t shared_at = (uint32_t)S * (uint32_t)a.H * 2u;
  auto src = [&](const Item<BL>& c, int i) {
    return c.start < 0 ? shared_at + (uint32_t)i * (uint32_t)a.Hs * 2u
                       : (uint32_t)p.sorted(c.start + i) * (uint32_t)a.H * 2u;
  };
  stream_items<WT, BL, NB, NS>(
      ring, w >> log_ks, R, nsh + hit, ks, KS, (uint64_t)a.a, item_of, src,
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
      int place[8];
      float sc[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = k0 + k < a.K && (ok >> (k0 + k) & 1);
        place[k] = in ? p.inverse(t * a.K + k0 + k) : -1;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sc[k] = a.before || place[k] < 0 ? 1.f : p.score(place[k]);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (place[k] >= 0) sum += row(place[k]) * sc[k];
    }
    if (nsh) sum += row(S + t) * p.gate(t);
    *(u32x2_t*)(a.out + (int64_t)t * a.D + row0 + 4 * d) =
        u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
  }
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

constexpr int kLds = 160 * 1024;

// MOST: the kernel's largest dynamic LDS (its static LDS beside it).
template <auto KERNEL, int MOST = kLds, class Args>
hipError_t launch_lds(dim3 grid, int lds, hipStream_t stream, const Args& a) {
  static const hipError_t attr_err =
      hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, MOST);
  if (attr_err != hipSuccess) return attr_err;
  return launch_k(false, KERNEL, grid, dim3(kThreads), lds, stream, a);
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

hipError_t launch_experts_fp4_many(DecodeArgs a, hipStream_t stream) {
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
  const uint32_t lds13 = sizeof(Labels) + a.smem_rows;
  hipError_t err = few ? launch_lds<decode_w13_kernel<WT, 1>>(grid, lds13, stream, a)
                       : launch_lds<decode_w13_kernel<WT, 4>>(grid, lds13, stream, a);
  if (err != hipSuccess) return err;
  a.log_ks = log_ks2;
  a.smem_rows = row_bytes(a.cap, std::max(a.H, a.Hs), log_ks2, U);
  grid = dim3(((a.Hs > 0) + hit) * nrb2);
  const uint32_t lds2 = sizeof(Labels) + a.smem_rows;
  return few ? launch_lds<decode_w2_kernel<WT, 1>, kLds / 2>(grid, lds2, stream, a)
             : launch_lds<decode_w2_kernel<WT, 4>, kLds / 2>(grid, lds2, stream, a);
}

template <int WT, int NB, int NS>
bool stream_w13(const DecodeArgs& a, hipStream_t stream, hipError_t& err) {
  const int lds = a.plan_lds + Ring<WT, kPairLoads<WT>, NB, NS>::kAll + kMeetRows * 1024;
  if (lds > kLds) return false;
  const int64_t pairs = (int64_t)std::min(a.E, a.T * a.K) * (a.H / 16) + a.Hs / 16;  // at the finest
  err = launch_lds<stream_w13_kernel<WT, NB, NS>>(dim3((unsigned)std::min<int64_t>(pairs, num_cus())), lds, stream, a);
  return true;
}

template <int WT, int BL, int NB, int NS>
bool stream_w2(DecodeArgs a, hipStream_t stream, hipError_t& err) {
  using Rg = Ring<WT, BL, NB, NS>;
  const int base = a.plan_lds + Rg::kAll;
  const int sums = (a.T * a.K + (a.Hs > 0 ? a.T : 0)) * Rg::kBlocks * 64;  // of one of KS shares
  if (base + sums > kLds) return false;
  a.log_ks = 0;
  while (a.log_ks < 3 && base + (sums << (a.log_ks + 1)) <= kLds) ++a.log_ks;
  err = launch_lds<stream_w2_kernel<WT, BL, NB, NS>>(dim3(ceil_div(a.D, BL * (WT == W_BF16 ? 8 : 16))),
                                                     base + (sums << a.log_ks), stream, a);
  return true;
}

// bf16.  Token rows per pass by the rows that an expert gets on average: a pass
// more streams its weights again, a larger one takes LDS from the ring.  The second
// product takes as few output rows per workgroup as give one workgroup per CU at
// most, where the slots' sums leave the room.
template <int BL>
bool w2_bf16(const DecodeArgs& a, int rows, hipStream_t stream, hipError_t& err) {
  if (rows <= 4)
    return stream_w2<W_BF16, BL, 1, BL == 1 ? 7 : BL == 2 ? 5 : 3>(a, stream, err) ||
           stream_w2<W_BF16, BL, 1, BL == 1 ? 4 : BL == 2 ? 3 : 2>(a, stream, err);
  if (rows <= 10)
    return stream_w2<W_BF16, BL, 2, BL == 1 ? 5 : BL == 2 ? 4 : 2>(a, stream, err) ||
           stream_w2<W_BF16, BL, 2, 2>(a, stream, err);
  return BL <= 2 && stream_w2<W_BF16, BL, 4, 2>(a, stream, err);
}

hipError_t launch_experts_bf16(const DecodeArgs& a, hipStream_t stream) {
  const int rows = a.T <= 8 ? 1 : ceil_div(a.T * a.K, a.E);
  hipError_t err = hipSuccess;
  if (rows <= 4) stream_w13<W_BF16, 1, 3>(a, stream, err);
  else if (rows <= 10) stream_w13<W_BF16, 2, 3>(a, stream, err) || stream_w13<W_BF16, 2, 2>(a, stream, err);
  else stream_w13<W_BF16, 4, 2>(a, stream, err);
  if (err != hipSuccess) return err;
  const int loads = ceil_div(a.D, 8 * num_cus());
  const bool ok = (loads <= 1 && w2_bf16<1>(a, rows, stream, err)) || (loads <= 2 && w2_bf16<2>(a, rows, stream, err)) ||
                  (loads <= 3 && w2_bf16<3>(a, rows, stream, err)) || w2_bf16<4>(a, rows, stream, err) ||
                  stream_w2<W_BF16, 2, 4, 2>(a, stream, err) || stream_w2<W_BF16, 2, 1, 2>(a, stream, err);
  return ok ? err : hipErrorInvalidValue;
}

// 4 bits.  The token rows of a stage take as much LDS as its weights, so the
// streams are for few rows; more share theirs between a workgroup's waves.
hipError_t launch_experts_fp4(const DecodeArgs& a, hipStream_t stream) {
  const int rows = a.T <= 4 ? 1 : ceil_div(a.T * a.K, a.E);
  if (rows > 4 || (a.Hs > 0 && a.T > 16)) return launch_experts_fp4_many(a, stream);
  hipError_t err = hipSuccess;
  if (rows <= 1) stream_w13<W_FP4, 1, 4>(a, stream, err);
  else stream_w13<W_FP4, 2, 3>(a, stream, err);
  if (err != hipSuccess) return err;
  const bool one = a.D / 16 <= num_cus();
  bool ok;
  if (rows <= 1)
    ok = (one && stream_w2<W_FP4, 1, 1, 5>(a, stream, err)) || (!one && stream_w2<W_FP4, 2, 1, 4>(a, stream, err)) ||
         stream_w2<W_FP4, 1, 2, 3>(a, stream, err);
  else
    ok = (!one && stream_w2<W_FP4, 2, 2, 3>(a, stream, err)) || stream_w2<W_FP4, 1, 2, 3>(a, stream, err);
  return ok ? err : hipErrorInvalidValue;
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

size_t al256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

size_t router_decode_workspace_bytes(int64_t T, int E) { return al256((size_t)T * E * 2); }

namespace {

hipError_t launch_logits(const RouterDecode& r, int T, int E, int D, hipStream_t stream) {
  const int rows = E + (r.w_gate != nullptr);
  const int tb = T >= 4 ? 4 : T >= 2 ? 2 : 1;
  const dim3 grid(ceil_div(rows, 4), ceil_div(T, tb));
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
// fp32 output rows, arrival counters.
size_t experts_decode_workspace_bytes(int64_t T, int64_t D, int64_t H, int K, int64_t Hs) {
  const int64_t S = T * K;
  return al256(PlanMap{(int)T, (int)S}.bytes()) + al256((size_t)(S * H + (Hs > 0 ? T * Hs : 0)) * 2) +
         al256((size_t)(S + (Hs > 0 ? T : 0)) * D * 4) + al256((size_t)(D / 32) * 4);
}

hipError_t launch_experts_decode(const ExpertsDecode& c, const RouterDecode* router, void* ws, hipStream_t stream) {
  DecodeArgs a{};
  a.T = c.T, a.D = c.D, a.H = c.H, a.E = c.E, a.K = c.K, a.Hs = c.Hs;
  a.x = (const bf16_t*)c.x;
  a.idx = c.idx, a.is64 = c.is64, a.before = c.before;
  a.scores = c.scores, a.limit = c.limit, a.gate = c.gate;
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
  p += al256((size_t)(S + Ts) * a.D * 4);
  a.count = (int*)p;
  a.out = (bf16_t*)c.out;

  PlanArgs pa{};
  pa.idx = c.idx, pa.is64 = c.is64, pa.scores = c.scores, pa.gate = c.gate;
  pa.T = a.T, pa.E = a.E, pa.K = a.K, pa.plan = (char*)ws;
  pa.count = a.count, pa.ncount = a.D / 32;
  hipError_t err;
  if (router) {
    err = launch_logits(*router, a.T, a.E, a.D, stream);
    if (err != hipSuccess) return err;
    select::GroupTopkArgs& t = pa.topk;
    t.z = router->logits;
    t.S = 1, t.T = a.T, t.E = a.E, t.K = a.K;
    t.aligned = ((uintptr_t)router->logits & 15) == 0;
    t.G = router->groups.groups, t.EG = a.E / t.G, t.kept = router->groups.kept, t.top2 = router->groups.top2;
    t.bias = router->bias;
    t.score_func = router->score_func, t.renorm = router->renorm, t.eps = router->eps, t.route_scale = router->scale;
    t.scores = router->top_scores, t.idx = router->top_idx;
    err = launch_plan_topk(pa, stream);
  } else {
    err = go_plan<0, 4>(pa, stream);
  }
  if (err != hipSuccess) return err;
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
  const dim3 grid(E * ceil_div(pairs, kWaves >> a.log_ks), offs ? std::min(tiles, 8) : tiles);
  return few ? launch_lds<grouped_mm_fp4_kernel<1>>(grid, a.smem_rows, stream, a)
             : launch_lds<grouped_mm_fp4_kernel<4>>(grid, a.smem_rows, stream, a);
}

}  // namespace ttamd
