// Group-limited selection of a token's experts in 64 bits (device functions;
// what it computes and why: router_group.hip).
#pragma once

#include "common.h"

namespace ttamd {
namespace select {

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

// p r + c with the constant in a scalar register pair (left to itself the
// compiler copies every constant of a Horner chain into vector registers
// first, three instructions a step instead of one).
__device__ __forceinline__ double fma_s(double p, double r, double c) {
  double d;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(p), "v"(r), "s"(c));
  return d;
}

// The larger and the smaller of two numbers (no NaN comes here; the builtins
// first canonicalise each operand, one more instruction apiece).
__device__ __forceinline__ double max_d(double a, double b) {
  double d;
  asm("v_max_f64 %0, %1, %2" : "=v"(d) : "v"(a), "v"(b));
  return d;
}
__device__ __forceinline__ double min_d(double a, double b) {
  double d;
  asm("v_min_f64 %0, %1, %2" : "=v"(d) : "v"(a), "v"(b));
  return d;
}

// The largest size of three numbers; NaN if one is.
__device__ __forceinline__ float most3(float a, float b, float c) {
  float d;
  asm("v_maximum3_f32 %0, |%1|, |%2|, |%3|" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

// exp(x), |x| <= 700.
__device__ __forceinline__ double exp_f64(double x) {
  // n = round(x / ln 2) by adding 1.5 * 2^52: n is then also the sum's low word
  const double magic = 6755399441055744.0;
  const double shifted = __builtin_fma(x, 1.4426950408889634, magic);
  const double n = shifted - magic;
  // ln 2 in two parts: floor(2^32 ln 2) / 2^32, whose product with n is exact,
  // and the rest
  double r = __builtin_fma(-n, 2977044471.0 / 4294967296.0, x);
  r = __builtin_fma(-n, 1.9082149292705877e-10, r);
  // the polynomial of degree 9 through e^r at the Chebyshev points of
  // [-ln2 / 2, ln2 / 2]: within 1.9e-14 of it
  double p = fma_s(0x1.72e107c874de9p-19, r, 0x1.a17df0d914d6cp-16);
  p = fma_s(p, r, 0x1.a01994c849582p-13);
  p = fma_s(p, r, 0x1.6c162bb7d965cp-10);
  p = fma_s(p, r, 0x1.11111123bf154p-7);
  p = fma_s(p, r, 0x1.55555588b8403p-5);
  p = fma_s(p, r, 0x1.5555555550d88p-3);
  p = fma_s(p, r, 0x1.ffffffffe74f1p-2);
  p = fma_s(p, r, 0x1.0000000000006p+0);
  p = fma_s(p, r, 0x1.000000000003dp+0);
  // times 2^n: |n| <= 1010 and 0.7 < p < 1.5, so the exponent field takes it
  const uint64_t b = as_u64(p);
  const uint32_t hi = (uint32_t)(b >> 32) + ((uint32_t)as_u64(shifted) << 20);
  return as_f64((uint64_t)hi << 32 | (uint32_t)b);
}

// 1 / d for 1 <= d <= 1.1e304: one Newton step from v_rcp_f64 (2^-23) gives
// 2^-45.
__device__ __forceinline__ double rcp_f64(double d) {
  const double y = __builtin_amdgcn_rcp(d);
  return __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
}

// Scores of single logits.  Exponents past 700 count as 700, a NaN as the
// least: the callers look for it themselves.
__device__ __forceinline__ double sigmoid_f64(float z) {
  return rcp_f64(1.0 + exp_f64(-(double)__builtin_amdgcn_fmed3f(z, -700.f, 700.f)));
}
__device__ __forceinline__ double exp_below(float z, float mx) {  // exp(z - mx), mx the row's maximum
  return exp_f64(max_d((double)z - (double)mx, -700.0));
}
// The same, NaN included.
__device__ __forceinline__ double score_of(float z, bool softmax, float mx, double inv) {
  const double s = softmax ? exp_below(z, mx) * inv : sigmoid_f64(z);
  return z == z ? s : __builtin_nan("");
}

// A selection value in the kernel's total order.
__device__ __forceinline__ double ordered(double v) {
  if (v != v) return as_f64(kNanKey);
  if (v == __builtin_inf()) return as_f64(kPosKey);
  if (v == -__builtin_inf()) return as_f64(kNegKey);
  return v;
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
  const uint64_t b = as_u64(v);
  const uint32_t hi = (uint32_t)(b >> 32);
  const uint32_t id = (uint32_t)e ^ (~(uint32_t)((int32_t)hi >> 31) & (uint32_t)kIdMask);  // kIdMask - e above zero
  return as_f64((uint64_t)hi << 32 | (((uint32_t)b & ~(uint32_t)kIdMask) | id));
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
  v = max_d(v, dpp_d<kDppXor1>(v));
  v = max_d(v, dpp_d<kDppXor2>(v));
  v = max_d(v, dpp_d<kDppHalfMirror>(v));
  v = max_d(v, dpp_d<kDppMirror>(v));
  if constexpr (LPT == 64) {
    double x, y;
    swap_halves_d<16>(v, x, y);
    v = max_d(x, y);
    swap_halves_d<32>(v, x, y);
    v = max_d(x, y);
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
__device__ __forceinline__ float all_sumf(float v) {
  return LPT == 64 ? wave64_sum(v) : row16_sum(v);
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
// ---- sorted lists of N keys per lane (descending; N a power of two) ----------
__device__ __forceinline__ void order2(double& hi, double& lo) {
  const double a = max_d(hi, lo), b = min_d(hi, lo);
  hi = a, lo = b;
}
// A list in any order (odd-even merge sort).
template <int N>
__device__ __forceinline__ void sort_list(double (&v)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j <= N - 1 - k; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k && i < N - j - k; ++i)
          if ((i + j) / (2 * p) == (i + j + k) / (2 * p)) order2(v[i + j], v[i + j + k]);
}
// The N largest of two sorted lists: the larger of a's i-th and b's i-th from
// the end form a bitonic sequence that holds them.
template <int N>
__device__ __forceinline__ void merge_lists(double (&a)[N], const double (&b)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = max_d(a[i], b[N - 1 - i]);
#pragma unroll
  for (int k = N / 2; k >= 1; k /= 2)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i & k) == 0) order2(a[i], a[i + k]);
}
template <int CTRL, int N>
__device__ __forceinline__ void merge_dpp(double (&a)[N]) {
  double b[N];
#pragma unroll
  for (int i = 0; i < N; ++i) b[i] = dpp_d<CTRL>(a[i]);
  merge_lists(a, b);
}
template <int DIST, int N>
__device__ __forceinline__ void merge_swap(double (&a)[N]) {
  double x[N], y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) swap_halves_d<DIST>(a[i], x[i], y[i]);
  merge_lists(x, y);
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = x[i];
}
// The token's N largest keys, sorted, in every lane.
template <int LPT, int N>
__device__ __forceinline__ void merge_lanes(double (&a)[N]) {
  merge_dpp<kDppXor1>(a);
  merge_dpp<kDppXor2>(a);
  merge_dpp<kDppHalfMirror>(a);
  merge_dpp<kDppMirror>(a);
  if constexpr (LPT == 64) {
    merge_swap<16>(a);
    merge_swap<32>(a);
  }
}

// How many of the 16 lanes of this lane's row hold a key above v.
template <int R>
__device__ __forceinline__ void count_above(double key, double v, int& n) {
  n += dpp_d<0x120 + R>(key) > v ? 1 : 0;  // row rotated by R
  if constexpr (R > 1) count_above<R - 1>(key, v, n);
}

// Merge the two best (a >= b) of two halves of a run.
__device__ __forceinline__ void merge2(double& a, double& b, double a2, double b2) {
  b = max_d(min_d(a, a2), max_d(b, b2));
  a = max_d(a, a2);
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

// Experts per lane with LPT lanes per token: every group an equal
// power-of-two run of the lanes.  0: the lanes cannot hold the groups.
inline int log2_ceil(int v) {
  int n = 0;
  while ((1 << n) < v) ++n;
  return n;
}
inline int experts_per_lane(int lpt, int G, int EG, int* log_run) {
  const int lg = log2_ceil(G), ll = log2_ceil(lpt);
  if (lg > ll) return 0;
  *log_run = ll - lg;
  return (EG + (1 << *log_run) - 1) >> *log_run;
}

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

// The picks of token t (its LPT lanes together): lane k < K gets pick k and its
// weight before route_scale.  `valid`: the lanes' token exists (t is in range
// regardless).  picked(i) runs once the picks are known, before the weights.
template <int LPT, int PL, int KL, int SRC, class Picked>
__device__ __forceinline__ void select_token(const GroupTopkArgs& a, int64_t t, bool valid, int& my_i, double& w,
                                             Picked picked) {
  const int gi = threadIdx.x & (LPT - 1);
  const int group = gi >> a.log_run;
  const int in0 = (gi & ((1 << a.log_run) - 1)) * a.per_lane;  // first place in the group
  const int n_live = group < a.G ? min(max(a.EG - in0, 0), a.per_lane) : 0;
  const int e0 = group * a.EG + in0;

  // Loads are unconditional, at indices clamped into the row (no branch
  // around each): whole 16-byte (bf16: 8-byte) loads where every lane's run of
  // experts is a multiple of 4.
  float z[PL];
  const bool quads = PL % 4 == 0 && a.aligned && (a.EG & 3) == 0 && (a.per_lane & 3) == 0;
  if (quads) {
    if constexpr (PL % 4 == 0) {
#pragma unroll
      for (int m = 0; m < PL; m += 4) {
        const int64_t at = t * a.E + min(e0 + m, a.E - 4);
        if constexpr (SRC == SRC_BF16) {
          const uint2 q = *(const uint2*)((const bf16_t*)a.z + at);
          z[m] = bf16_to_f32(q.x & 0xffff), z[m + 1] = bf16_to_f32(q.x >> 16);
          z[m + 2] = bf16_to_f32(q.y & 0xffff), z[m + 3] = bf16_to_f32(q.y >> 16);
        } else {
          // (a vector, not a struct of floats, whose loads would be merged with the other
          // branch's into 16 single ones: 16384 tokens of 256 experts, traced, 15.6 us so, 20.6)
          floatx4_t q = *(const floatx4_t*)((const float*)a.z + at);
          if constexpr (SRC == SRC_PARTIALS) {
            for (int s = 1; s < a.S; ++s) {
              q += *(const floatx4_t*)((const float*)a.z + at + (int64_t)s * a.T * a.E);
            }
            q = floatx4_t{round_bf16(q[0]), round_bf16(q[1]), round_bf16(q[2]), round_bf16(q[3])};
          }
          z[m] = q[0], z[m + 1] = q[1], z[m + 2] = q[2], z[m + 3] = q[3];
        }
      }
    }
  } else {
#pragma unroll
    for (int m = 0; m < PL; ++m) z[m] = logit_at<SRC>(a, t, min(e0 + m, a.E - 1));
  }
  float bias[PL];
  if (a.bias) {
#pragma unroll
    for (int m = 0; m < PL; ++m) bias[m] = a.bias[min(e0 + m, a.E - 1)];
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
  float mx = 0.f, nan = 0.f;  // nan: NaN when a logit is (or softmax has no finite maximum)
  double inv = 1.0;
  // is any logit or bias of the wave's tokens NaN or infinite?
  float size = 0.f;
#pragma unroll
  for (int m = 0; m < PL; m += 2) size = most3(z[m], z[m + 1], size);
  if (a.bias) {
#pragma unroll
    for (int m = 0; m < PL; m += 2) size = most3(bias[m], bias[m + 1], size);
  }
  const bool special = __builtin_amdgcn_ballot_w64(!(size < INFINITY)) != 0;
  if (special) {
#pragma unroll
    for (int m = 0; m < PL; ++m) nan += z[m] == z[m] ? 0.f : z[m];
  }
  if (a.score_func == 0) {
    mx = -INFINITY;
#pragma unroll
    for (int m = 0; m < PL; ++m) mx = fmaxf(mx, z[m]);  // (a clamped index repeats a logit of the row)
    mx = all_maxf<LPT>(mx);
    if (special) {
      if (!__builtin_isfinite(mx)) nan = __builtin_nanf("");  // inf - inf
      nan = all_sumf<LPT>(nan);                               // one NaN makes the whole row NaN
    }
    double sum = 0.0;
#pragma unroll
    for (int m = 0; m < PL; ++m) {
      const double x = exp_below(z[m], mx);
      v[m] = m < n_live ? x : 0.0;
      sum += v[m];
    }
    inv = rcp_f64(all_sum<LPT>(sum));
#pragma unroll
    for (int m = 0; m < PL; ++m) v[m] *= inv;
  } else {
#pragma unroll
    for (int m = 0; m < PL; ++m) v[m] = sigmoid_f64(z[m]);
  }
  if (a.bias) {
#pragma unroll
    for (int m = 0; m < PL; ++m) v[m] += (double)bias[m];
  }
  // NaN and infinities take the general order; numbers are in it already
  if (special) {
#pragma unroll
    for (int m = 0; m < PL; ++m) {
      const bool bad = a.score_func == 0 ? nan != nan : z[m] != z[m];
      v[m] = ordered(bad ? __builtin_nan("") : v[m]);
    }
  }

  // keys; slots without an expert: the high word alone makes them the least
  auto kill = [](double d) { return as_f64((uint64_t)kDeadHi << 32 | (uint32_t)as_u64(d)); };
#pragma unroll
  for (int m = 0; m < PL; ++m) v[m] = with_id(v[m], e0 + m);
  if (a.per_lane < PL || a.EG != a.per_lane << a.log_run || a.G << a.log_run != LPT) {  // uniform
#pragma unroll
    for (int m = 0; m < PL; ++m) v[m] = m < n_live ? v[m] : kill(v[m]);
  }
  const double dead = as_f64((uint64_t)kDeadHi << 32);

  // the lane's KL best
  double top[KL];
#pragma unroll
  for (int i = 0; i < KL; ++i) top[i] = i < PL ? v[i] : dead;
  sort_list(top);
#pragma unroll
  for (int c = KL; c < PL; c += KL) {
    double more[KL];
#pragma unroll
    for (int i = 0; i < KL; ++i) more[i] = c + i < PL ? v[c + i] : dead;
    sort_list(more);
    merge_lists(top, more);
  }

  if (a.kept < a.G) {  // uniform
    // (without the ids: groups of equal values are equal)
    double b1 = as_f64(as_u64(top[0]) & ~kIdMask), b2 = as_f64(as_u64(top[1]) & ~kIdMask);
    run_top2<LPT>(b1, b2, 1 << a.log_run);
    double value = (a.top2 && a.EG > 1) ? group_sum(b1, b2) : b1;
    value = group < a.G ? with_id(value, group) : dead;
    bool in = false;
    if (LPT == 16 || a.log_run >= 2) {  // uniform
      // a group is kept if fewer than `kept` groups are above it, counted over
      // a row's 16 lanes (LPT 64: every fourth lane's value, which meets every
      // group equally often)
      double key = value;
      int shift = a.log_run;
      if constexpr (LPT == 64) {
        const uint64_t b = as_u64(value);
        const int from = 16 * (gi & 15);  // byte address of lane 4 (gi % 16)
        const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)b);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(b >> 32));
        key = as_f64((uint64_t)hi << 32 | lo);
        shift = a.log_run - 2;
      }
      int above = key > value ? 1 : 0;
      count_above<15>(key, value, above);
      in = above < (a.kept << shift);
    } else {
      for (int r = 0; r < a.kept; ++r) {
        const double best = all_max<LPT>(value);
        if (value == best) {
          in = true;
          value = dead;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < KL; ++i) top[i] = in ? top[i] : kill(top[i]);
  }
  // the token's
  merge_lanes<LPT>(top);
  double mine = top[0];
#pragma unroll
  for (int i = 1; i < KL; ++i) mine = gi == i ? top[i] : mine;
  // K picks fit the kept groups, so no dead key is among the first K; the
  // clamp only keeps the index in range regardless
  my_i = min(id_of(mine), a.E - 1);
  picked(my_i);
  // lane k's pick: its unbiased score again from its logit (one exponential,
  // instead of every expert's score kept through the selection)
  w = 0.0;
  if (gi < a.K) {
    w = score_of(logit_at<SRC>(a, t, my_i), a.score_func == 0, mx, inv);
    if (a.score_func == 0 && nan != nan) w = __builtin_nan("");
  }
  if (a.renorm) {
    const double total = all_sum<LPT>(w) + (double)a.eps;
    w = w / total;
  }
}

}  // namespace select
}  // namespace ttamd
