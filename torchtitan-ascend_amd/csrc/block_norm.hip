// The norms before and after a block, fused with its gate, its residual scale
// and (for expert rows) the K-way combine, forward and backward, on MI355X.
//
//   f = sum_k prob[t, k] * rows[inverse[t K + k]]   (K = 1: the branch itself)
//   p = f * r_f * w_post,   r_f = 1 / sqrt(mean f^2 + eps)     (no w_post: p = f)
//   u = residual + scale * act(gate) * p
//   n = u * r_u * w_pre,    r_u = 1 / sqrt(mean u^2 + eps)
//
// Everything is computed in fp32 from the inputs and rounded once, where it is
// stored; n is taken from the unrounded u.
//
// Memory-bound.  A workgroup takes a row at a time, 8 consecutive columns (16
// bytes of bf16) per thread and vector, so a row is read once into registers,
// both mean squares are reductions of those registers, and u and n leave from
// them.  The rows of a workgroup are walked with its columns' weights in
// registers and the next row's loads in flight.  Measured (bf16): 8192 rows of
// 5120, forward 56 us (6.0 TB/s of rows in and out), backward 92 us (5.5 TB/s)
// and its column sums 7; of 2048, 28 and 49 us; one row of 7168 4.0 us, a
// launch; the combine of eight gathered rows of 2048, 8192 tokens, 68 us (5.4
// TB/s).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "gemm_common.h"
#include "kernels.h"

namespace ttamd {
namespace {

enum GateKind { GATE_NONE = 0, GATE_TOKEN = 1, GATE_CHANNEL = 2, GATE_FULL = 3 };

// 8 consecutive elements of bf16 or fp32, as loaded.
struct Raw8 {
  uint4 a, b;  // b: the upper half of fp32
};
__device__ __forceinline__ Raw8 fetch8(const void* p, int64_t i, bool f32) {
  Raw8 r;
  if (f32) {
    const uint4* q = (const uint4*)((const float*)p + i);
    r.a = load_stream(q), r.b = load_stream(q + 1);
  } else {
    r.a = load_stream((const uint4*)((const bf16_t*)p + i));
    r.b = make_uint4(0u, 0u, 0u, 0u);
  }
  return r;
}
__device__ __forceinline__ void widen8(const Raw8& r, bool f32, float* v) {
  if (f32) {
    v[0] = __uint_as_float(r.a.x), v[1] = __uint_as_float(r.a.y), v[2] = __uint_as_float(r.a.z);
    v[3] = __uint_as_float(r.a.w), v[4] = __uint_as_float(r.b.x), v[5] = __uint_as_float(r.b.y);
    v[6] = __uint_as_float(r.b.z), v[7] = __uint_as_float(r.b.w);
  } else {
    unpack8(r.a, v);
  }
}
// The same for weights: cached loads.
__device__ __forceinline__ void load8(const void* p, int64_t i, bool f32, float* v) {
  Raw8 r;
  const uint4* q = f32 ? (const uint4*)((const float*)p + i) : (const uint4*)((const bf16_t*)p + i);
  r.a = q[0];
  r.b = f32 ? q[1] : q[0];
  widen8(r, f32, v);
}
__device__ __forceinline__ void store8(void* p, int64_t i, bool f32, const float* v) {
  if (f32) {
    float4* q = (float4*)((float*)p + i);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *(uint4*)((bf16_t*)p + i) = pack8(v);
  }
}
__device__ __forceinline__ float load1(const void* p, int64_t i, bool f32) {
  return f32 ? ((const float*)p)[i] : bf16_to_f32(((const bf16_t*)p)[i]);
}
__device__ __forceinline__ Raw8 no_raw() {
  Raw8 r;
  r.a = r.b = make_uint4(0u, 0u, 0u, 0u);
  return r;
}

// Sums over the workgroup, in every thread, in wave order; `phase` alternates
// between two sets of slots, so one barrier per sum is enough.
template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float (*slots)[N][16], int& phase) {
  const int w = threadIdx.x >> 6, nw = blockDim.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave64_sum(v[i]);
  if (nw == 1) return;
  float (*s)[16] = slots[phase & 1];
  ++phase;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i][w] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float t = s[i][0];
    for (int k = 1; k < nw; ++k) t += s[i][k];
    v[i] = t;
  }
}

// ---------------------------------------------------------------------------
// Forward: one vector per thread.  COMBINE: the first kCombineRows expert rows
// of the next token are in flight while this one is reduced, and its row ids
// one token earlier still (scalar loads: a token is a workgroup's), so a
// gathered row waits for neither.  A ninth row and later ones are fetched when
// they are needed: 8192 tokens of 2048, 8 rows each 69 us (5.4 TB/s), 10 rows
// 86 (5.1), 16 rows 136 (4.7).
// ---------------------------------------------------------------------------
constexpr int kCombineRows = 8;
typedef const __attribute__((address_space(4))) int cint_t;  // read only while the kernel runs: scalar loads
typedef const __attribute__((address_space(4))) float cfloat_t;

template <bool S32, bool COMBINE, int GATE>
__global__ __launch_bounds__(1024) void norm_forward_kernel(const NormArgs a) {
  __shared__ float slots[2][1][16];
  constexpr int KR = COMBINE ? kCombineRows : 1;
  int phase = 0;
  const int D = a.D;
  const int col = 8 * threadIdx.x;
  const bool on = col < D;
  // w_post * scale * act(channel gate), and w_pre
  float wu[8], wn[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) wu[j] = 1.f, wn[j] = 0.f;
  const float inv_d = 1.f / (float)D;
  const int last_row = a.T * a.K - 1;

  Raw8 q_r = no_raw(), q_g = no_raw();
  uint4 q_f[KR];
  float q_p[KR];
  int q_id[KR];  // rows of the token fetched next
#pragma unroll
  for (int k = 0; k < KR; ++k) q_f[k] = make_uint4(0u, 0u, 0u, 0u), q_p[k] = 1.f, q_id[k] = 0;
  auto row_at = [&](int slot) {  // the row of slot t K + k
    return a.inverse ? min(max(((cint_t*)a.inverse)[slot], 0), last_row) : slot;
  };
  auto fetch_ids = [&](int t) {
    if constexpr (COMBINE) {
#pragma unroll
      for (int k = 0; k < KR; ++k)
        if (k < a.K) q_id[k] = row_at(t * a.K + k);
    }
  };
  auto fetch = [&](int t) {
    const int64_t at = (int64_t)t * D + col;
    if constexpr (COMBINE) {
#pragma unroll
      for (int k = 0; k < KR; ++k) {
        if (k < a.K) {  // uniform
          if (a.probs) q_p[k] = ((cfloat_t*)a.probs)[t * a.K + k];
          if (on) q_f[k] = load_stream((const uint4*)(a.rows + (int64_t)q_id[k] * D + col));
        }
      }
    }
    if (!on) return;
    if (!COMBINE && a.rows) q_f[0] = load_stream((const uint4*)(a.rows + at));
    if (a.residual) q_r = fetch8(a.residual, at, S32);
    if constexpr (GATE == GATE_FULL) q_g = fetch8(a.gate, at, a.gate32);
  };
  const int step = gridDim.x;
  int t = blockIdx.x;
  if (t < a.T) {
    fetch_ids(t);
    fetch(t);
    fetch_ids(min(t + step, a.T - 1));
  }
  if (on) {
    if (a.post) load8(a.post, col, a.post32, wu);
    if (a.pre) load8(a.pre, col, a.pre32, wn);
    if constexpr (GATE == GATE_CHANNEL) {
      float g[8];
      load8(a.gate, col, a.gate32, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) wu[j] *= a.sigmoid ? sigmoid_f(g[j]) : g[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) wu[j] *= a.scale;
  for (; t < a.T; t += step) {
    float x[8], r[8];  // x: f, then u
    if constexpr (COMBINE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.f;
#pragma unroll
      for (int k = 0; k < KR; ++k) {
        if (k < a.K) {
          float w[8];
          unpack8(q_f[k], w);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = fmaf(q_p[k], w[j], x[j]);
        }
      }
    } else {
      unpack8(q_f[0], x);
    }
    widen8(q_r, S32, r);
    float g[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = 1.f;
    if constexpr (GATE == GATE_FULL) widen8(q_g, a.gate32, g);
    if constexpr (GATE == GATE_TOKEN) g[0] = load1(a.gate, t, a.gate32);
    if (t + step < a.T) {
      fetch(t + step);
      fetch_ids(min(t + 2 * step, a.T - 1));
    }
    if constexpr (COMBINE) {
      for (int k = KR; k < a.K; ++k) {  // more choices than are kept in flight
        const int slot = t * a.K + k;
        const float p = a.probs ? a.probs[slot] : 1.f;
        if (on) {
          float w[8];
          unpack8(load_stream((const uint4*)(a.rows + (int64_t)row_at(slot) * D + col)), w);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = fmaf(p, w[j], x[j]);
        }
      }
    }
    if constexpr (GATE == GATE_FULL) {
      if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = sigmoid_f(g[j]);
      }
    }
    if constexpr (GATE == GATE_TOKEN) {
      if (a.sigmoid) g[0] = sigmoid_f(g[0]);
    }
    float rf = 1.f;
    if (a.post) {
      float s[1] = {0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] = fmaf(x[j], x[j], s[0]);
      block_sums<1>(s, slots, phase);
      rf = 1.f / sqrtf(s[0] * inv_d + a.eps);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float w = GATE == GATE_TOKEN ? g[0] * wu[j] : GATE == GATE_FULL ? g[j] * wu[j] : wu[j];
      x[j] = a.rows ? r[j] + w * (x[j] * rf) : r[j];
    }
    const int64_t at = (int64_t)t * D + col;
    if (a.u && on) store8(a.u, at, S32, x);
    float ru = 1.f;
    if (a.pre) {
      float s[1] = {0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] = fmaf(x[j], x[j], s[0]);
      if (!on) s[0] = 0.f;
      block_sums<1>(s, slots, phase);
      ru = 1.f / sqrtf(s[0] * inv_d + a.eps);
      if (on) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x[j] * ru * wn[j];
        store8(a.n, at, false, v);
      }
    }
    if (a.rstd && threadIdx.x == 0) {
      a.rstd[t] = rf;
      a.rstd[a.T + t] = ru;
    }
  }
}

// ---------------------------------------------------------------------------
// Backward.  u is recomputed from the branch, the residual and the saved
// r_f, so the gradient is of exactly what the forward computed.  With a the
// gate's act and fh = f r_f:
//   q = dn * w_pre;       dU = du + r_u (q - u r_u^2 mean(q u))
//   dresidual = dU;       dw_pre = sum_t dn u r_u
//   dgate = scale w_post act' dU fh   (summed over what it was broadcast)
//   dw_post = sum_t scale a dU fh
//   q2 = scale a w_post dU;  df = r_f (q2 - f r_f^2 mean(q2 f))
// A gate per channel (or none) is the same for every token, so dgate and
// dw_post are then one column sum, S = sum_t dU fh, times factors that the
// second launch applies.  The column sums of a workgroup's rows stay in
// registers and leave once per workgroup as partial sums, which that launch
// adds in workgroup order (no atomics: the same bits every time).
// ---------------------------------------------------------------------------
template <bool S32, int GATE, int MAX_THREADS>
__global__ __launch_bounds__(MAX_THREADS) void norm_backward_kernel(const NormBwdArgs a) {
  __shared__ float slots1[2][1][16], slots2[2][2][16];
  int ph1 = 0, ph2 = 0;
  const NormArgs& f = a.fwd;
  const int D = f.D;
  const int col = 8 * threadIdx.x;
  const bool on = col < D;
  float wu[8], wn[8];  // scale * w_post * act(channel gate), and w_pre
  float s_f[8], s_n[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) wu[j] = 1.f, wn[j] = 0.f, s_f[j] = 0.f, s_n[j] = 0.f;
  const float inv_d = 1.f / (float)D;
  Raw8 q_f = no_raw(), q_r = no_raw(), q_u = no_raw(), q_n = no_raw(), q_g = no_raw();
  float q_rf = 1.f, q_ru = 1.f, q_t = 1.f;
  auto fetch = [&](int t) {
    q_rf = f.rstd[t], q_ru = f.rstd[f.T + t];
    if constexpr (GATE == GATE_TOKEN) q_t = load1(f.gate, t, f.gate32);
    if (!on) return;
    const int64_t at = (int64_t)t * D + col;
    if (f.rows) q_f = fetch8(f.rows, at, false);
    if (f.residual) q_r = fetch8(f.residual, at, S32);
    if (a.du) q_u = fetch8(a.du, at, S32);
    if (a.dn) q_n = fetch8(a.dn, at, false);
    if constexpr (GATE == GATE_FULL) q_g = fetch8(f.gate, at, f.gate32);
  };
  int t = blockIdx.x;
  if (t < f.T) fetch(t);  // in flight before the weights are waited for
  if (on) {
    if (f.post) load8(f.post, col, f.post32, wu);
    if (f.pre) load8(f.pre, col, f.pre32, wn);
    if constexpr (GATE == GATE_CHANNEL) {
      float g[8];
      load8(f.gate, col, f.gate32, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) wu[j] *= f.sigmoid ? sigmoid_f(g[j]) : g[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) wu[j] *= f.scale;
  for (; t < f.T; t += gridDim.x) {
    const int64_t at = (int64_t)t * D + col;
    float x[8], u[8], g[8], dn[8], act[GATE == GATE_FULL ? 8 : 1];  // g: du, then dU
    widen8(q_f, false, x);
    widen8(q_r, S32, u);
    widen8(q_u, S32, g);
    widen8(q_n, false, dn);
    const float rf = q_rf, ru = q_ru;
    act[0] = 1.f;
    if constexpr (GATE == GATE_FULL) widen8(q_g, f.gate32, act);
    if constexpr (GATE == GATE_TOKEN) act[0] = q_t;
    if (GATE >= GATE_TOKEN && GATE != GATE_CHANNEL && f.sigmoid) {
#pragma unroll
      for (int j = 0; j < (GATE == GATE_FULL ? 8 : 1); ++j) act[j] = sigmoid_f(act[j]);
    }
    auto gate = [&](int j) { return act[GATE == GATE_FULL ? j : 0]; };
    if (t + (int)gridDim.x < f.T) fetch(t + gridDim.x);
    if (f.rows) {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] += gate(j) * wu[j] * (x[j] * rf);
    }
    if (f.pre) {
      float s[1] = {0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] = fmaf(dn[j] * wn[j], u[j], s[0]);
      block_sums<1>(s, slots1, ph1);
      const float c = s[0] * inv_d * ru * ru;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s_n[j] = fmaf(dn[j], u[j] * ru, s_n[j]);
        g[j] += ru * (dn[j] * wn[j] - u[j] * c);
      }
    }
    if (a.dresidual && on) store8(a.dresidual, at, S32, g);
    if (!f.rows) continue;  // uniform
    float s[2] = {0.f, 0.f};  // sum of q2 f, sum of dgate
    float dg[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float gf = g[j] * (x[j] * rf), av = gate(j);
      s_f[j] = fmaf(av, gf, s_f[j]);
      if constexpr (GATE == GATE_TOKEN || GATE == GATE_FULL) {
        dg[j] = gf * wu[j] * (f.sigmoid ? av * (1.f - av) : 1.f);
        s[1] += dg[j];
      }
      g[j] *= av * wu[j];
      s[0] = fmaf(g[j], x[j], s[0]);
    }
    if (GATE == GATE_FULL && a.dgate && on) store8(a.dgate, at, f.gate32, dg);
    if (f.post || GATE == GATE_TOKEN) block_sums<2>(s, slots2, ph2);
    const float c = f.post ? s[0] * inv_d * rf * rf : 0.f;
    if (on && a.dbranch) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = rf * (g[j] - x[j] * c);
      store8(a.dbranch, at, false, v);
    }
    if (GATE == GATE_TOKEN && a.dgate && threadIdx.x == 0) {
      if (f.gate32) ((float*)a.dgate)[t] = s[1];
      else ((bf16_t*)a.dgate)[t] = (bf16_t)f32_to_bf16(s[1]);
    }
  }
  // partial sums of this workgroup's rows: [2][grid][D]
  if (on) {
    float* part = a.part + (int64_t)blockIdx.x * D;
    if (a.dpost || (GATE == GATE_CHANNEL && a.dgate)) store8(part, col, true, s_f);
    if (a.dpre) store8(part + (int64_t)gridDim.x * D, col, true, s_n);
  }
}

// The n partial rows of each column added in a fixed order: 64 runs of rows
// side by side, 8 loads of each in flight, then the runs pairwise (16 in a
// wave's lanes, then the four waves); and the factors that turn S into dw_post
// and the channel gate's gradient.  A workgroup takes 16 columns; blockIdx.y:
// 0 S, 1 dw_pre.
__device__ __forceinline__ void store4(void* out, int c, bool f32, const float4& s) {
  if (f32)
    *(float4*)((float*)out + c) = s;
  else
    *(uint2*)((bf16_t*)out + c) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
}
__global__ __launch_bounds__(256) void column_sum_kernel(const NormBwdArgs a, int n) {
  __shared__ float4 sh[4][4];
  const NormArgs& f = a.fwd;
  const bool channel = a.dgate && f.gate_kind == GATE_CHANNEL;
  if (blockIdx.y == 0 ? !(a.dpost || channel) : !a.dpre) return;
  const int cx = threadIdx.x & 3, ry = threadIdx.x >> 2;
  const int c = (blockIdx.x * 4 + cx) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < f.D) {
    const float* p = a.part + (int64_t)blockIdx.y * n * f.D + c;
#pragma unroll 8
    for (int r = ry; r < n; r += 64) {
      const float4 v = *(const float4*)(p + (int64_t)r * f.D);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
#pragma unroll
  for (int d = 4; d < 64; d *= 2) {
    s.x += __shfl_xor(s.x, d, kWave), s.y += __shfl_xor(s.y, d, kWave);
    s.z += __shfl_xor(s.z, d, kWave), s.w += __shfl_xor(s.w, d, kWave);
  }
  if ((threadIdx.x & 63) < 4) sh[threadIdx.x >> 6][cx] = s;
  __syncthreads();
  if (ry != 0 || c >= f.D) return;
#pragma unroll
  for (int r = 1; r < 4; ++r) {
    const float4 v = sh[r][cx];
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  if (blockIdx.y == 1) return store4(a.dpre, c, f.pre32, s);
  const float sum[4] = {s.x, s.y, s.z, s.w};
  float dp[4], dg[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float act = 1.f, dact = 1.f;
    if (f.gate_kind == GATE_CHANNEL) {
      act = load1(f.gate, c + j, f.gate32);
      if (f.sigmoid) {
        act = sigmoid_f(act);
        dact = act * (1.f - act);
      }
    }
    dp[j] = f.scale * act * sum[j];
    dg[j] = f.scale * (f.post ? load1(f.post, c + j, f.post32) : 1.f) * dact * sum[j];
  }
  if (a.dpost) store4(a.dpost, c, f.post32, make_float4(dp[0], dp[1], dp[2], dp[3]));
  if (channel) store4(a.dgate, c, f.gate32, make_float4(dg[0], dg[1], dg[2], dg[3]));
}

int round64(int v) { return (v + 63) & ~63; }

// Workgroups that a call takes at most: `waves` waves per CU, at least `least`
// workgroups of them.
int64_t most_groups(int D, int waves, int least) {
  return (int64_t)num_cus() * std::max(least, waves * 64 / round64(D / 8));
}
// ... and the number that spreads T rows evenly over no more than that.
int even_groups(int64_t T, int64_t most) {
  const int64_t per = (T + most - 1) / most;
  return (int)((T + per - 1) / per);
}
// Measured (bf16, us): 8192 rows of 5120, 16 / 24 / 32 waves 61 / 55 / 65; of
// 7168 with one / two workgroups per CU 88 / 77; combine, eight rows of 2048
// per token, 8192 tokens, 8 / 12 / 24 waves 72 / 70 / 76.
int forward_groups(int64_t T, int D, bool combine) {
  return even_groups(T, combine ? most_groups(D, 12, 1) : most_groups(D, 24, 2));
}
// Every workgroup of the backward leaves two rows of partial sums, so with few
// rows it takes four or more, down to one workgroup per CU (1003 rows of 2056:
// 32 -> 27 us).  8192 rows of 2048, 8 / 12 / 24 waves: 56 / 51 / 58 us.
int64_t backward_most(int64_t T, int D) {
  return std::min(most_groups(D, 12, 1), std::max<int64_t>(num_cus(), T / 4));
}

template <bool S32, bool COMBINE>
hipError_t go_forward(const NormArgs& a, hipStream_t stream) {
  const int threads = round64(a.D / 8);
  const dim3 grid(forward_groups(a.T, a.D, COMBINE));
  switch (a.gate_kind) {
    case GATE_TOKEN:
      return launch_k(false, norm_forward_kernel<S32, COMBINE, GATE_TOKEN>, grid, dim3(threads), 0, stream, a);
    case GATE_CHANNEL:
      return launch_k(false, norm_forward_kernel<S32, COMBINE, GATE_CHANNEL>, grid, dim3(threads), 0, stream, a);
    case GATE_FULL:
      return launch_k(false, norm_forward_kernel<S32, COMBINE, GATE_FULL>, grid, dim3(threads), 0, stream, a);
    default:
      return launch_k(false, norm_forward_kernel<S32, COMBINE, GATE_NONE>, grid, dim3(threads), 0, stream, a);
  }
}

template <bool S32>
hipError_t go_backward(const NormBwdArgs& b, int groups, hipStream_t stream) {
  const dim3 block(round64(b.fwd.D / 8));
  switch (b.fwd.gate_kind) {
    case GATE_TOKEN:
      return launch_k(false, norm_backward_kernel<S32, GATE_TOKEN, 1024>, dim3(groups), block, 0, stream, b);
    case GATE_CHANNEL:
      return launch_k(false, norm_backward_kernel<S32, GATE_CHANNEL, 1024>, dim3(groups), block, 0, stream, b);
    case GATE_FULL:
      // (a gate per element needs a few registers more than 1024 threads leave)
      if (block.x <= 512)
        return launch_k(false, norm_backward_kernel<S32, GATE_FULL, 512>, dim3(groups), block, 0, stream, b);
      return launch_k(false, norm_backward_kernel<S32, GATE_FULL, 1024>, dim3(groups), block, 0, stream, b);
    default:
      return launch_k(false, norm_backward_kernel<S32, GATE_NONE, 1024>, dim3(groups), block, 0, stream, b);
  }
}

}  // namespace

hipError_t launch_norm_forward(const NormArgs& a, hipStream_t stream) {
  if (a.T == 0) return hipSuccess;
  const bool combine = a.rows && (a.K > 1 || a.inverse || a.probs);
  if (a.stream32) return combine ? go_forward<true, true>(a, stream) : go_forward<true, false>(a, stream);
  return combine ? go_forward<false, true>(a, stream) : go_forward<false, false>(a, stream);
}

// Two planes of partial sums of as many workgroups as any call of at most T
// rows takes.
size_t norm_backward_workspace_bytes(int64_t T, int64_t D) {
  return 2 * (size_t)std::min(T, backward_most(T, (int)D)) * (size_t)D * sizeof(float);
}

hipError_t launch_norm_backward(const NormBwdArgs& b, hipStream_t stream) {
  const NormArgs& a = b.fwd;
  // (no rows: no partial sums either, and the column sums are zeros)
  const int groups = a.T == 0 ? 0 : even_groups(a.T, backward_most(a.T, a.D));
  hipError_t err = hipSuccess;
  if (a.T > 0) err = a.stream32 ? go_backward<true>(b, groups, stream) : go_backward<false>(b, groups, stream);
  if (err != hipSuccess || !(b.dpost || b.dpre || (b.dgate && a.gate_kind == GATE_CHANNEL))) return err;
  return launch_k(false, column_sum_kernel, dim3((a.D + 15) / 16, 2), dim3(256), 0, stream, b, groups);
}

}  // namespace ttamd
