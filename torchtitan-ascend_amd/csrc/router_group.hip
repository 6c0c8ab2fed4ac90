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
// cycles, as v_fma_f32 does).  Exponential and reciprocal are good to 2^-45,
// eight times finer than the values' 2^-42 that the selection compares.
//
// Layout: LPT lanes per token (16: four tokens per wave; 64: one).  Every
// group owns an equal power-of-two run of lanes and every lane up to PL
// consecutive experts of it, so a group's best two meet in log2(run) exchange
// steps and no lane straddles two groups.  Each value and its expert are packed
// into one double: the low 10 mantissa bits (2^-42 of the value) hold the id, so
// plain maxima and minima order values, ties and identities at once.  A lane
// sorts its K best with a sorting network; lists then merge pairwise across
// the token's lanes (16 lanes: 4 merges, in the VALU's own lane exchanges), in
// place of K dependent rounds of a maximum over all lanes (16384 tokens of 256
// experts: 19.0 -> 15.6 us, one token 5.4 -> 3.8).  A lane's first two are also
// its share of its group's value.
//
// What bounds it: few tokens, the latency of one launch (4 us); many tokens,
// VALU issue (1140 instructions per wave of four tokens at E = 256, K = 8: 8 of
// 13.6 us at 16384 tokens in a stream of launches), not the logits' bytes (3.4 us).  The bias is 4 of
// the 13.6: a load per expert and lane, 88 instructions.  On the gate GEMM's
// partials, with the histogram, 22 us.
#include <type_traits>

#include "common.h"
#include "gemm_common.h"
#include "kernels.h"
#include "router_select.h"

namespace ttamd {
namespace {

using namespace select;

template <int LPT, int PL, int KL, int SRC>
__global__ __launch_bounds__(256) void group_topk_kernel(const GroupTopkArgs a) {
  constexpr int TPB = 256 / LPT;
  const int gi = threadIdx.x & (LPT - 1);
  const int64_t t_own = (int64_t)blockIdx.x * TPB + threadIdx.x / LPT;
  const bool valid = t_own < a.T;
  const int64_t t = valid ? t_own : a.T - 1;
  const bool out = gi < a.K;
  int my_i;
  double w;
  select_token<LPT, PL, KL, SRC>(a, t, valid, my_i, w, [&](int pick) {
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
          atomicAdd(&lh[min(max(c, 0), 1) * a.E + pick], 1);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * a.E; i += 256) {
          const int n = lh[i], c = c0 + i / a.E;
          if (n > 0 && c < a.nchunks) atomicAdd(&a.hist[(int64_t)(i % a.E) * a.nchunks + c], n);
        }
      }
    }
  });
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
// The differences cancel (a renormalised weight near 1, a softmax score near
// 1), so scores and sums are 64-bit as in the forward, and dz is rounded once.
// Lane k holds pick k; only softmax needs a score per expert.  LPT lanes per
// token, each a run of 4 experts of every 4 LPT: whole 16-byte (bf16: 8-byte)
// stores where E % 4 == 0.  An index outside [0, E) contributes nothing; one
// that occurs twice adds twice.
// Bound by the launch up to a few thousand tokens (softmax, 256 experts: 32
// tokens 6.4 us, 4096 7.1), then by VALU issue (16384 16.1 us, of which 1489
// instructions per wave take 10; sigmoid, without the scores of the other
// experts, 11.0 and 6; the bytes alone 6.9).
// ---------------------------------------------------------------------------
struct TopkBwdArgs {
  const float* grad;   // [T, K]
  const int64_t* idx;  // [T, K]
  const void* z;       // [T, E]
  int T, E, K;
  int score_func, renorm;
  float eps, route_scale;
  void* dz;            // [T, E] in z's type
  int aligned;         // dz starts at a multiple of 16 bytes
};

template <int LPT, int PL, bool BF16>
__global__ __launch_bounds__(256) void topk_backward_kernel(const TopkBwdArgs a) {
  constexpr int TPB = 256 / LPT;
  const int gi = threadIdx.x & (LPT - 1);
  const int64_t t_own = (int64_t)blockIdx.x * TPB + threadIdx.x / LPT;
  const bool valid = t_own < a.T;
  const int64_t t = valid ? t_own : a.T - 1;
  auto eid = [&](int m) { return 4 * gi + (m & 3) + 4 * LPT * (m >> 2); };
  auto logit = [&](int e) {
    return BF16 ? bf16_to_f32(((const bf16_t*)a.z)[t * a.E + e]) : ((const float*)a.z)[t * a.E + e];
  };
  // this lane's pick
  int my_e = -1;
  double g = 0.0;
  if (gi < a.K) {
    const int64_t e = a.idx[t * a.K + gi];
    if (e >= 0 && e < a.E) {
      my_e = (int)e;
      g = (double)a.grad[t * a.K + gi] * (double)a.route_scale;
    }
  }
  const float my_z = logit(max(my_e, 0));

  double s[PL];  // softmax: the scores
  double w;      // the pick's score
  if (a.score_func == 0) {
    float z[PL], mx = -INFINITY;
#pragma unroll
    for (int m = 0; m < PL; ++m) {
      z[m] = logit(min(eid(m), a.E - 1));
      mx = fmaxf(mx, z[m]);  // (a repeated last one changes no maximum)
    }
    mx = all_maxf<LPT>(mx);
    double sum = 0.0;
#pragma unroll
    for (int m = 0; m < PL; ++m) {
      const double x = score_of(z[m], true, mx, 1.0);
      s[m] = eid(m) < a.E ? x : 0.0;
      sum += s[m];
    }
    const double inv = __builtin_isfinite(mx) ? rcp_f64(all_sum<LPT>(sum)) : __builtin_nan("");
#pragma unroll
    for (int m = 0; m < PL; ++m) s[m] *= inv;
    w = score_of(my_z, true, mx, inv);
  } else {
    w = score_of(my_z, false, 0.f, 1.0);
  }
  if (my_e < 0) w = 0.0;
  double d = g;
  if (a.renorm) {
    const double S = all_sum<LPT>(w) + (double)a.eps, gs = all_sum<LPT>(g * w);
    d = (g - gs / S) / S;
  }
  if (my_e < 0) d = 0.0;
  double dot = 0.0;
  if (a.score_func == 0) dot = all_sum<LPT>(d * w);
  else d *= w * (1.0 - w);

  // the picks' terms to the lanes of their experts, in pick order
  double acc[PL];
#pragma unroll
  for (int m = 0; m < PL; ++m) acc[m] = 0.0;
  const int base = lane_id() & ~(LPT - 1);  // lanes of this token in the wave
  for (int k = 0; k < a.K; ++k) {
    const int ek = __shfl(my_e, base + k, kWave);
    const double dk = __shfl(d, base + k, kWave);
#pragma unroll
    for (int m = 0; m < PL; ++m) acc[m] += eid(m) == ek ? dk : 0.0;
  }
  if (!valid) return;
  const bool quads = (a.E & 3) == 0 && a.aligned;
#pragma unroll
  for (int m = 0; m < PL; m += 4) {
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (float)(a.score_func == 0 ? s[m + i] * (acc[m + i] - dot) : acc[m + i]);
    const int64_t at = t * a.E + eid(m);
    if (quads) {
      if (eid(m) < a.E) {
        if constexpr (BF16)
          *(uint2*)((bf16_t*)a.dz + at) = make_uint2(pack_bf16x2(r[0], r[1]), pack_bf16x2(r[2], r[3]));
        else
          *(float4*)((float*)a.dz + at) = make_float4(r[0], r[1], r[2], r[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (eid(m + i) < a.E) {
          if constexpr (BF16)
            ((bf16_t*)a.dz)[at + i] = (bf16_t)f32_to_bf16(r[i]);
          else
            ((float*)a.dz)[at + i] = r[i];
        }
      }
    }
  }
}

template <int LPT, int PL, int KL>
hipError_t go_source(int src, const GroupTopkArgs& a, hipStream_t stream) {
  constexpr int TPB = 256 / LPT;
  const dim3 grid((unsigned)((a.T + TPB - 1) / TPB));
  if (src == SRC_F32) return launch_k(false, group_topk_kernel<LPT, PL, KL, SRC_F32>, grid, dim3(256), 0, stream, a);
  if (src == SRC_BF16) return launch_k(false, group_topk_kernel<LPT, PL, KL, SRC_BF16>, grid, dim3(256), 0, stream, a);
  return launch_k(false, group_topk_kernel<LPT, PL, KL, SRC_PARTIALS>, grid, dim3(256), 0, stream, a);
}
template <int LPT, int PL>
hipError_t go_group(int src, const GroupTopkArgs& a, hipStream_t stream) {
  return a.K <= 8 ? go_source<LPT, PL, 8>(src, a, stream) : go_source<LPT, PL, 16>(src, a, stream);
}

hipError_t launch_group_topk(int src, GroupTopkArgs a, hipStream_t stream) {
  // 16 lanes per token while they hold at most 4 experts each, and wherever
  // issue slots count; a wave per token in between, whose lists are shorter
  // to build.  Measured (us, 16 lanes / 64): E = 256, 8 groups, 1024 tokens
  // 6.4 / 4.4, 2048 6.5 / 5.6, 4096 6.6 / 8.0, 16384 13.6 / 23.1; E = 160,
  // 1024 5.6 / 4.5, 2048 5.7 / 5.9; E = 64, 32 tokens 3.6 / 4.2.
  int lr16 = 0, lr64 = 0;
  const int p16 = experts_per_lane(16, a.G, a.EG, &lr16), p64 = experts_per_lane(64, a.G, a.EG, &lr64);
  const bool narrow = p16 > 0 && p16 <= 16 && (p16 <= 4 || a.T > 160 * p16);
  a.log_run = narrow ? lr16 : lr64;
  a.per_lane = narrow ? p16 : p64;
  if (narrow) {
    if (p16 <= 4) return go_group<16, 4>(src, a, stream);
    if (p16 <= 8) return go_group<16, 8>(src, a, stream);
    if (p16 <= 12) return go_group<16, 12>(src, a, stream);
    return go_group<16, 16>(src, a, stream);
  }
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
  a.aligned = ((uintptr_t)grad_logits & 15) == 0;
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
