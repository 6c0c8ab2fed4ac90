// Router selection limited to groups of experts, and the gradient of the
// routing weights with respect to the logits, on MI355X (gfx950).
//
//   s = softmax(z) or sigmoid(z);  v = s + bias          (E experts, G groups)
//   value of a group = sum of its two largest v, or its largest
//   keep the `kept` groups of largest value (ties: lower group); pick the K
//   experts of the kept groups in descending v (ties: lower id)
//   w_k = s[idx_k];  renorm: w_k /= sum_k w_k + eps;  w_k *= route_scale
//
// Scores and selection values are 64-bit floats.  Two candidates closer than
// a 32-bit ulp are common (256 sigmoid scores + bias: about one token in 10^4
// at every rank), and a 32-bit value would then pick by its own rounding; a
// double costs the same VALU cycles here (a 64-lane v_fma_f64 issues in four
// cycles, as v_fma_f32 does).  The exponential is a degree-11 Taylor sum on
// [-ln2 / 2, ln2 / 2] (remainder below 1e-14), the reciprocal two Newton
// steps from v_rcp_f64.
//
// Layout: LPT lanes per token (16: four tokens per wave; 64: one).  Every
// group owns an equal power-of-two run of lanes and every lane up to PL
// consecutive experts of it, so a group's best two meet in log2(run) exchange
// steps and no lane straddles two groups.  A lane packs each value and its
// expert into one double: the low 10 mantissa bits (2^-42 of the value) hold
// the id, so one max over the lanes finds the winner, its lower-id tie rule
// and its identity at once.
//
// What bounds it: few tokens, the latency of one launch and of K dependent
// rounds; many tokens, VALU issue (about 1100 instructions per wave of four
// tokens at E = 256, K = 8), not the logits' bytes.
#include <type_traits>

#include "common.h"
#include "gemm_common.h"
#include "kernels.h"

namespace ttamd {
namespace {

constexpr int kGroupWaveTokens = 2048;
constexpr int kIdBits = 10;
constexpr uint64_t kIdMask = (1u << kIdBits) - 1;
// Order of values that are not finite numbers: NaN first, then +inf, the
// numbers (at most 3.4e38 in size), -inf, then slots that cannot be picked.
constexpr uint64_t kNanKey = 0x7fe8000000000000ull;
constexpr uint64_t kPosKey = 0x7fd0000000000000ull;
constexpr uint64_t kNegKey = 0xffd0000000000000ull;
constexpr uint32_t kDeadHi = 0xffefffffu;

__device__ __forceinline__ double as_f64(uint64_t b) { return __builtin_bit_cast(double, b); }
__device__ __forceinline__ uint64_t as_u64(double d) { return __builtin_bit_cast(uint64_t, d); }

// exp(x) for -745 <= x <= 700 (clamped; NaN stays NaN).
__device__ __forceinline__ double exp_f64(double x) {
  x = x < -745.0 ? -745.0 : (x > 700.0 ? 700.0 : x);
  const double n = x == x ? __builtin_rint(x * 1.4426950408889634) : 0.0;  // defined as an int below
  // ln 2 in two parts: floor(2^32 ln 2) / 2^32, whose product with n is exact,
  // and the rest
  double r = __builtin_fma(-n, 2977044471.0 / 4294967296.0, x);
  r = __builtin_fma(-n, 1.9082149292705877e-10, r);
  double p = 1.0 / 39916800.0;
  p = __builtin_fma(p, r, 1.0 / 3628800.0);
  p = __builtin_fma(p, r, 1.0 / 362880.0);
  p = __builtin_fma(p, r, 1.0 / 40320.0);
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}

// 1 / d for 1 <= d <= 1.1e304, or NaN.
__device__ __forceinline__ double rcp_f64(double d) {
  double y = __builtin_amdgcn_rcp(d);
  y = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
  return __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
}

__device__ __forceinline__ double sigmoid_f64(double z) { return rcp_f64(1.0 + exp_f64(-z)); }

// A selection value in the kernel's total order.
__device__ __forceinline__ double ordered(double v) {
  if (v != v) return as_f64(kNanKey);
  if (v == __builtin_inf()) return as_f64(kPosKey);
  if (v == -__builtin_inf()) return as_f64(kNegKey);
  return v + 0.0;  // -0 becomes +0
}

// a >= b, both ordered(): the group's value as the sum of the two.
__device__ __forceinline__ double group_sum(double a, double b) {
  const double nan = as_f64(kNanKey), pos = as_f64(kPosKey), neg = as_f64(kNegKey);
  double s = a + b;
  s = (b == neg) ? neg : s;
  s = (a == pos) ? (b == neg ? nan : pos) : s;
  return a == nan ? nan : s;
}

// The value with its expert's id in the low bits: of equal values the lower
// id is the larger key, on either side of zero.
__device__ __forceinline__ double with_id(double v, int e) {
  const uint64_t b = as_u64(v) & ~kIdMask;
  return as_f64(b | ((b >> 63) ? (uint64_t)e : kIdMask - (uint64_t)e));
}
__device__ __forceinline__ int id_of(double key) {
  const uint64_t b = as_u64(key);
  return (int)((b >> 63) ? (b & kIdMask) : kIdMask - (b & kIdMask));
}

template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  const uint64_t b = as_u64(v);
  const uint32_t lo = (uint32_t)dpp_i<CTRL>((int)(uint32_t)b), hi = (uint32_t)dpp_i<CTRL>((int)(b >> 32));
  return as_f64((uint64_t)hi << 32 | lo);
}

template <int DIST>
__device__ __forceinline__ void swap_halves_d(double v, double& x, double& y) {
  const uint64_t b = as_u64(v);
  uint32_t xl, yl, xh, yh;
  swap_halves<DIST>((uint32_t)b, xl, yl);
  swap_halves<DIST>((uint32_t)(b >> 32), xh, yh);
  x = as_f64((uint64_t)xh << 32 | xl);
  y = as_f64((uint64_t)yh << 32 | yl);
}

// Reductions over a token's LPT lanes; every lane gets the result.
template <int LPT>
__device__ __forceinline__ double all_max(double v) {
  v = __builtin_fmax(v, dpp_d<kDppXor1>(v));
  v = __builtin_fmax(v, dpp_d<kDppXor2>(v));
  v = __builtin_fmax(v, dpp_d<kDppHalfMirror>(v));
  v = __builtin_fmax(v, dpp_d<kDppMirror>(v));
  if constexpr (LPT == 64) {
    double x, y;
    swap_halves_d<16>(v, x, y);
    v = __builtin_fmax(x, y);
    swap_halves_d<32>(v, x, y);
    v = __builtin_fmax(x, y);
  }
  return v;
}
template <int LPT>
__device__ __forceinline__ double all_sum(double v) {
  v += dpp_d<kDppXor1>(v);
  v += dpp_d<kDppXor2>(v);
  v += dpp_d<kDppHalfMirror>(v);
  v += dpp_d<kDppMirror>(v);
  if constexpr (LPT == 64) {
    double x, y;
    swap_halves_d<16>(v, x, y);
    v = x + y;
    swap_halves_d<32>(v, x, y);
    v = x + y;
  }
  return v;
}
template <int LPT>
__device__ __forceinline__ float all_maxf(float v) {
  v = row16_max(v);
  if constexpr (LPT == 64) {
    uint32_t x, y;
    swap_halves<16>(__float_as_uint(v), x, y);
    v = fmaxf(__uint_as_float(x), __uint_as_float(y));
    swap_halves<32>(__float_as_uint(v), x, y);
    v = fmaxf(__uint_as_float(x), __uint_as_float(y));
  }
  return v;
}
template <int LPT>
__device__ __forceinline__ float all_sumf(float v) {
  return LPT == 64 ? wave64_sum(v) : row16_sum(v);
}
template <int LPT>
__device__ __forceinline__ int all_min(int v) {
  v = min(v, dpp_i<kDppXor1>(v));
  v = min(v, dpp_i<kDppXor2>(v));
  v = min(v, dpp_i<kDppHalfMirror>(v));
  v = min(v, dpp_i<kDppMirror>(v));
  if constexpr (LPT == 64) {
    uint32_t x, y;
    swap_halves<16>((uint32_t)v, x, y);
    v = min((int)x, (int)y);
    swap_halves<32>((uint32_t)v, x, y);
    v = min((int)x, (int)y);
  }
  return v;
}

// Merge the two best (a >= b) of two halves of a run.
__device__ __forceinline__ void merge2(double& a, double& b, double a2, double b2) {
  b = __builtin_fmax(__builtin_fmin(a, a2), __builtin_fmax(b, b2));
  a = __builtin_fmax(a, a2);
}
// The two best of every aligned run of `run` lanes (a power of two, uniform).
template <int LPT>
__device__ __forceinline__ void run_top2(double& a, double& b, int run) {
  if (run > 1) merge2(a, b, dpp_d<kDppXor1>(a), dpp_d<kDppXor1>(b));
  if (run > 2) merge2(a, b, dpp_d<kDppXor2>(a), dpp_d<kDppXor2>(b));
  if (run > 4) merge2(a, b, dpp_d<kDppHalfMirror>(a), dpp_d<kDppHalfMirror>(b));
  if (run > 8) merge2(a, b, dpp_d<kDppMirror>(a), dpp_d<kDppMirror>(b));
  if constexpr (LPT == 64) {
    double ax, ay, bx, by;
    if (run > 16) {
      swap_halves_d<16>(a, ax, ay);
      swap_halves_d<16>(b, bx, by);
      a = ax, b = bx;
      merge2(a, b, ay, by);
    }
    if (run > 32) {
      swap_halves_d<32>(a, ax, ay);
      swap_halves_d<32>(b, bx, by);
      a = ax, b = bx;
      merge2(a, b, ay, by);
    }
  }
}

enum LogitSource { SRC_F32 = 0, SRC_BF16 = 1, SRC_PARTIALS = 2 };

struct GroupTopkArgs {
  const void* z;      // logits [T, E] (fp32 or bf16), or partial sums [S][T][E] fp32
  int S, T, E, K;
  int aligned;        // z starts at a multiple of 16 bytes
  int G, EG, kept;    // groups, experts of each, groups kept
  int log_run;        // log2 of the lanes of a group
  int per_lane;       // experts per lane (<= PL)
  int top2;           // group value: sum of two largest, else the largest
  const float* bias;  // [E] or null
  int score_func;     // 0 softmax, 1 sigmoid
  int renorm;
  float eps, route_scale;
  float* scores;      // [T, K]
  int64_t* idx;       // [T, K]
  bf16_t* logits;     // SRC_PARTIALS: [T, E] or null
  int* hist;          // SRC_PARTIALS: the route histogram or null
  int nchunks, chunk;
};

template <int SRC>
__device__ __forceinline__ float logit_at(const GroupTopkArgs& a, int64_t t, int e) {
  if constexpr (SRC == SRC_F32) return ((const float*)a.z)[t * a.E + e];
  if constexpr (SRC == SRC_BF16) return bf16_to_f32(((const bf16_t*)a.z)[t * a.E + e]);
  // the gate GEMM's slices, summed in slice order; the Linear's output is bf16
  const float* p = (const float*)a.z + t * a.E + e;
  float z = p[0];
  for (int s = 1; s < a.S; ++s) z += p[(int64_t)s * a.T * a.E];
  return round_bf16(z);
}

template <int LPT, int PL, int SRC>
__global__ __launch_bounds__(256) void group_topk_kernel(const GroupTopkArgs a) {
  constexpr int TPB = 256 / LPT;
  const int gi = threadIdx.x & (LPT - 1);
  const int64_t t_own = (int64_t)blockIdx.x * TPB + threadIdx.x / LPT;
  const bool valid = t_own < a.T;
  const int64_t t = valid ? t_own : a.T - 1;
  const int group = gi >> a.log_run;
  const int in0 = (gi & ((1 << a.log_run) - 1)) * a.per_lane;  // first place in the group
  const int n_live = group < a.G ? min(max(a.EG - in0, 0), a.per_lane) : 0;
  const int e0 = group * a.EG + in0;

  float z[PL];
  // whole 16-byte loads where every lane's run of experts is a multiple of 4
  const bool quads = SRC != SRC_BF16 && PL % 4 == 0 && a.aligned && (a.EG & 3) == 0 && (a.per_lane & 3) == 0;
  if (quads) {
    if constexpr (PL % 4 == 0) {
      const float* row = (const float*)a.z + t * a.E + e0;
#pragma unroll
      for (int m = 0; m < PL; m += 4) {
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (m < n_live) {
          q = *(const float4*)(row + m);
          if constexpr (SRC == SRC_PARTIALS) {
            for (int s = 1; s < a.S; ++s) {
              const float4 p = *(const float4*)(row + (int64_t)s * a.T * a.E + m);
              q.x += p.x, q.y += p.y, q.z += p.z, q.w += p.w;
            }
            q.x = round_bf16(q.x), q.y = round_bf16(q.y), q.z = round_bf16(q.z), q.w = round_bf16(q.w);
          }
        }
        z[m] = q.x, z[m + 1] = q.y, z[m + 2] = q.z, z[m + 3] = q.w;
      }
    }
  } else {
#pragma unroll
    for (int m = 0; m < PL; ++m) z[m] = m < n_live ? logit_at<SRC>(a, t, e0 + m) : 0.f;
  }
  if constexpr (SRC == SRC_PARTIALS) {
    if (a.logits && valid) {
#pragma unroll
      for (int m = 0; m < PL; ++m)
        if (m < n_live) a.logits[t * a.E + e0 + m] = (bf16_t)f32_to_bf16(z[m]);
    }
  }

  // scores, then selection values
  double v[PL];
  float mx = 0.f;
  double inv = 1.0;
  if (a.score_func == 0) {
    mx = -INFINITY;
#pragma unroll
    for (int m = 0; m < PL; ++m) mx = fmaxf(mx, m < n_live ? z[m] : -INFINITY);
    mx = all_maxf<LPT>(mx);
    double sum = 0.0;
#pragma unroll
    for (int m = 0; m < PL; ++m) {
      v[m] = m < n_live ? exp_f64((double)z[m] - (double)mx) : 0.0;
      sum += v[m];
    }
    inv = rcp_f64(all_sum<LPT>(sum));
#pragma unroll
    for (int m = 0; m < PL; ++m) v[m] *= inv;
  } else {
#pragma unroll
    for (int m = 0; m < PL; ++m) v[m] = sigmoid_f64((double)z[m]);
  }
#pragma unroll
  for (int m = 0; m < PL; ++m) {
    if (a.bias) v[m] += m < n_live ? (double)a.bias[e0 + m] : 0.0;
    v[m] = ordered(v[m]);
  }

  const double dead = as_f64((uint64_t)kDeadHi << 32);
  bool keep = n_live > 0;
  if (a.kept < a.G) {  // uniform
    double b1 = dead, b2 = dead;
#pragma unroll
    for (int m = 0; m < PL; ++m) {
      const double x = m < n_live ? v[m] : dead;
      b2 = __builtin_fmax(b2, __builtin_fmin(b1, x));
      b1 = __builtin_fmax(b1, x);
    }
    run_top2<LPT>(b1, b2, 1 << a.log_run);
    double value = (a.top2 && a.EG > 1) ? group_sum(b1, b2) : b1;
    if (group >= a.G) value = dead;
    bool in = false;
    for (int r = 0; r < a.kept; ++r) {
      const double best = all_max<LPT>(value);
      const int win = all_min<LPT>(value == best ? group : LPT);
      if (group == win) {
        in = true;
        value = dead;
      }
    }
    keep = keep && in;
  }
#pragma unroll
  for (int m = 0; m < PL; ++m) v[m] = (keep && m < n_live) ? with_id(v[m], e0 + m) : dead;

  int my_i = 0;
  for (int k = 0; k < a.K; ++k) {
    double best = v[0];
#pragma unroll
    for (int m = 1; m < PL; ++m) best = __builtin_fmax(best, v[m]);
    best = all_max<LPT>(best);
    // K picks fit the kept groups, so a live key is left in every round; the
    // clamp only keeps the index in range regardless
    if (gi == k) my_i = min(id_of(best), a.E - 1);
#pragma unroll
    for (int m = 0; m < PL; ++m) {
      const uint64_t b = as_u64(v[m]);
      const uint32_t hi = v[m] == best ? kDeadHi : (uint32_t)(b >> 32);
      v[m] = as_f64((uint64_t)hi << 32 | (uint32_t)b);
    }
  }

  const bool out = gi < a.K;
  if constexpr (SRC == SRC_PARTIALS) {
    if (a.hist) {
      // the workgroup's TPB * K flat slots span at most two chunks: counted
      // in LDS, then one atomic per nonzero (expert, chunk)
      __shared__ int lh[2 * 256];
      const int c0 = (int)(((int64_t)blockIdx.x * TPB * a.K) / a.chunk);
      for (int i = threadIdx.x; i < 2 * a.E; i += 256) lh[i] = 0;
      __syncthreads();
      if (out && valid) {
        const int c = (int)((t * a.K + gi) / a.chunk) - c0;
        atomicAdd(&lh[min(max(c, 0), 1) * a.E + my_i], 1);
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * a.E; i += 256) {
        const int n = lh[i], c = c0 + i / a.E;
        if (n > 0 && c < a.nchunks) atomicAdd(&a.hist[(int64_t)(i % a.E) * a.nchunks + c], n);
      }
    }
  }
  // lane k's pick: its unbiased score again from its logit (one exponential,
  // instead of every expert's score kept through the selection)
  double w = 0.0;
  if (out) {
    const double zi = (double)logit_at<SRC>(a, t, my_i);
    w = a.score_func == 0 ? exp_f64(zi - (double)mx) * inv : sigmoid_f64(zi);
  }
  if (a.renorm) {
    const double total = all_sum<LPT>(w) + (double)a.eps;
    w = w / total;
  }
  if (out && valid) {
    a.scores[t * a.K + gi] = (float)(w * (double)a.route_scale);
    a.idx[t * a.K + gi] = my_i;
  }
}

// ---------------------------------------------------------------------------
// Gradient of the routing weights: d(top_scores) [T, K] -> d(logits) [T, E].
// The selection has no gradient, so groups and bias do not enter:
//   g_k = route_scale * grad[k];  S = sum_k s[idx_k] + eps
//   ds_k = renorm ? g_k / S - (sum_j g_j s[idx_j]) / S^2 : g_k
//   softmax: dz = s * (ds - sum_k ds_k s[idx_k]);  sigmoid: dz = ds s (1 - s)
// 32-bit arithmetic (every step is smooth).  LPT lanes per token, lane i the
// experts i, i + LPT, ...: coalesced.  An index outside [0, E) matches no
// expert; one that occurs twice adds twice.  One pass over the logits.
// ---------------------------------------------------------------------------
struct TopkBwdArgs {
  const float* grad;   // [T, K]
  const int64_t* idx;  // [T, K]
  const void* z;       // [T, E]
  int T, E, K;
  int score_func, renorm;
  float eps, route_scale;
  void* dz;            // [T, E] in z's type
};

template <int LPT, int PL, bool BF16>
__global__ __launch_bounds__(256) void topk_backward_kernel(const TopkBwdArgs a) {
  constexpr int TPB = 256 / LPT;
  const int gi = threadIdx.x & (LPT - 1);
  const int64_t t_own = (int64_t)blockIdx.x * TPB + threadIdx.x / LPT;
  const bool valid = t_own < a.T;
  const int64_t t = valid ? t_own : a.T - 1;
  float s[PL], d[PL];
  float mx = -INFINITY;
#pragma unroll
  for (int m = 0; m < PL; ++m) {
    const int e = gi + m * LPT;
    s[m] = -INFINITY;
    if (e < a.E)
      s[m] = BF16 ? bf16_to_f32(((const bf16_t*)a.z)[t * a.E + e]) : ((const float*)a.z)[t * a.E + e];
    mx = fmaxf(mx, s[m]);
    d[m] = 0.f;
  }
  if (a.score_func == 0) {
    mx = all_maxf<LPT>(mx);
    float sum = 0.f;
#pragma unroll
    for (int m = 0; m < PL; ++m) {
      s[m] = gi + m * LPT < a.E ? expf(s[m] - mx) : 0.f;
      sum += s[m];
    }
    const float inv = 1.f / all_sumf<LPT>(sum);
#pragma unroll
    for (int m = 0; m < PL; ++m) s[m] *= inv;
  } else {
#pragma unroll
    for (int m = 0; m < PL; ++m) s[m] = 1.f / (1.f + expf(-s[m]));
  }
  // the lanes' picks: lane k holds pick k (K <= 16 <= LPT)
  int64_t my = -1;
  float g = 0.f;
  if (gi < a.K) {
    my = a.idx[t * a.K + gi];
    g = a.grad[t * a.K + gi] * a.route_scale;
  }
  const int my_e = (my >= 0 && my < a.E) ? (int)my : -1;
  // lanes of this token in the wave
  const int base = lane_id() & ~(LPT - 1);
  float S = 0.f, gs = 0.f;
  if (a.renorm) {
    for (int k = 0; k < a.K; ++k) {
      const int ek = __shfl(my_e, base + k, kWave);
      const float gk = __shfl(g, base + k, kWave);
      float v = 0.f;
#pragma unroll
      for (int m = 0; m < PL; ++m) v = gi + m * LPT == ek ? s[m] : v;
      v = all_sumf<LPT>(v);  // one lane holds s[ek]
      S += v;
      gs += gk * v;
    }
    S += a.eps;
  }
  const float sub = a.renorm ? gs / (S * S) : 0.f;
  for (int k = 0; k < a.K; ++k) {
    const int ek = __shfl(my_e, base + k, kWave);
    const float gk = __shfl(g, base + k, kWave);
    const float dk = a.renorm ? gk / S - sub : gk;
#pragma unroll
    for (int m = 0; m < PL; ++m) d[m] += gi + m * LPT == ek ? dk : 0.f;
  }
  float dot = 0.f;
  if (a.score_func == 0) {
#pragma unroll
    for (int m = 0; m < PL; ++m) dot += d[m] * s[m];
    dot = all_sumf<LPT>(dot);
  }
  if (!valid) return;
#pragma unroll
  for (int m = 0; m < PL; ++m) {
    const int e = gi + m * LPT;
    if (e >= a.E) continue;
    const float r = a.score_func == 0 ? s[m] * (d[m] - dot) : d[m] * s[m] * (1.f - s[m]);
    if constexpr (BF16)
      ((bf16_t*)a.dz)[t * a.E + e] = (bf16_t)f32_to_bf16(r);
    else
      ((float*)a.dz)[t * a.E + e] = r;
  }
}

int log2_ceil(int v) {
  int n = 0;
  while ((1 << n) < v) ++n;
  return n;
}

template <int LPT, int PL>
hipError_t go_group(int src, const GroupTopkArgs& a, hipStream_t stream) {
  constexpr int TPB = 256 / LPT;
  const dim3 grid((unsigned)((a.T + TPB - 1) / TPB));
  if (src == SRC_F32) return launch_k(false, group_topk_kernel<LPT, PL, SRC_F32>, grid, dim3(256), 0, stream, a);
  if (src == SRC_BF16) return launch_k(false, group_topk_kernel<LPT, PL, SRC_BF16>, grid, dim3(256), 0, stream, a);
  return launch_k(false, group_topk_kernel<LPT, PL, SRC_PARTIALS>, grid, dim3(256), 0, stream, a);
}

// Experts per lane with LPT lanes per token: every group an equal
// power-of-two run of the lanes.  0: the lanes cannot hold the groups.
int experts_per_lane(int lpt, int G, int EG, int* log_run) {
  const int lg = log2_ceil(G), ll = log2_ceil(lpt);
  if (lg > ll) return 0;
  *log_run = ll - lg;
  return (EG + (1 << *log_run) - 1) >> *log_run;
}

hipError_t launch_group_topk(int src, GroupTopkArgs a, hipStream_t stream) {
  // A wave per token while there are few tokens (its chain of rounds is
  // short), four tokens per wave where issue slots count.
  int lr16 = 0, lr64 = 0;
  const int p16 = experts_per_lane(16, a.G, a.EG, &lr16), p64 = experts_per_lane(64, a.G, a.EG, &lr64);
  const bool narrow = p16 > 0 && p16 <= 16 && a.T > kGroupWaveTokens;
  a.log_run = narrow ? lr16 : lr64;
  a.per_lane = narrow ? p16 : p64;
  if (narrow) {
    if (p16 <= 2) return go_group<16, 2>(src, a, stream);
    if (p16 <= 4) return go_group<16, 4>(src, a, stream);
    if (p16 <= 8) return go_group<16, 8>(src, a, stream);
    if (p16 <= 12) return go_group<16, 12>(src, a, stream);
    return go_group<16, 16>(src, a, stream);
  }
  if (p64 <= 2) return go_group<64, 2>(src, a, stream);
  if (p64 <= 4) return go_group<64, 4>(src, a, stream);
  if (p64 <= 8) return go_group<64, 8>(src, a, stream);
  if (p64 <= 16) return go_group<64, 16>(src, a, stream);
  return go_group<64, 32>(src, a, stream);  // E <= 1024, G <= 64: at most 32 per lane
}

}  // namespace

hipError_t launch_router_topk_grouped(const void* logits, bool bf16, const float* bias, int T, int E, int K,
                                      const RouterGroups& g, int score_func, int renorm, float renorm_eps,
                                      float route_scale, float* top_scores, int64_t* top_idx, hipStream_t stream) {
  if (T == 0) return hipSuccess;
  GroupTopkArgs a = {};
  a.z = logits;
  a.S = 1, a.T = T, a.E = E, a.K = K;
  a.aligned = ((uintptr_t)logits & 15) == 0;
  a.G = g.groups, a.EG = E / g.groups, a.kept = g.kept, a.top2 = g.top2;
  a.bias = bias;
  a.score_func = score_func, a.renorm = renorm, a.eps = renorm_eps, a.route_scale = route_scale;
  a.scores = top_scores, a.idx = top_idx;
  return launch_group_topk(bf16 ? SRC_BF16 : SRC_F32, a, stream);
}

hipError_t launch_group_topk_partials(const float* part, int S, const float* bias, int T, int E, int K,
                                      const RouterGroups& g, int score_func, int renorm, float renorm_eps,
                                      float route_scale, float* top_scores, int64_t* top_idx, void* logits, int* hist,
                                      int nchunks, int chunk, hipStream_t stream) {
  GroupTopkArgs a = {};
  a.z = part;
  a.S = S, a.T = T, a.E = E, a.K = K;
  a.aligned = 1;  // a workspace
  a.G = g.groups, a.EG = E / g.groups, a.kept = g.kept, a.top2 = g.top2;
  a.bias = bias;
  a.score_func = score_func, a.renorm = renorm, a.eps = renorm_eps, a.route_scale = route_scale;
  a.scores = top_scores, a.idx = top_idx, a.logits = (bf16_t*)logits;
  a.hist = hist, a.nchunks = nchunks, a.chunk = chunk;
  return launch_group_topk(SRC_PARTIALS, a, stream);
}

hipError_t launch_router_topk_backward(const float* grad, const int64_t* idx, const void* logits, bool bf16, int T,
                                       int E, int K, int score_func, int renorm, float renorm_eps, float route_scale,
                                       void* grad_logits, hipStream_t stream) {
  if (T == 0) return hipSuccess;
  TopkBwdArgs a = {};
  a.grad = grad, a.idx = idx, a.z = logits, a.T = T, a.E = E, a.K = K;
  a.score_func = score_func, a.renorm = renorm, a.eps = renorm_eps, a.route_scale = route_scale;
  a.dz = grad_logits;
  auto go = [&](auto lpt, auto pl) {
    constexpr int LPT = decltype(lpt)::value, PL = decltype(pl)::value;
    const dim3 grid((unsigned)((T + 256 / LPT - 1) / (256 / LPT)));
    if (bf16) return launch_k(false, topk_backward_kernel<LPT, PL, true>, grid, dim3(256), 0, stream, a);
    return launch_k(false, topk_backward_kernel<LPT, PL, false>, grid, dim3(256), 0, stream, a);
  };
  const std::integral_constant<int, 16> l16{};
  const std::integral_constant<int, 64> l64{};
  if (E <= 64) return go(l16, std::integral_constant<int, 4>{});
  if (E <= 128) return go(l16, std::integral_constant<int, 8>{});
  if (E <= 256) return go(l16, std::integral_constant<int, 16>{});
  return go(l64, std::integral_constant<int, 16>{});
}

}  // namespace ttamd
