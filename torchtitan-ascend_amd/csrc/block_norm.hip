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
// Memory-bound: a row is read once into registers (8 consecutive columns per
// 16-byte vector, VPT vectors per thread), both mean squares are reductions of
// those registers, and u and n leave from them.  Up to 2048 columns a wave
// holds a row and no barrier is needed; wider rows (and few rows, where the
// latency of one counts) take a workgroup each.  A workgroup walks rows with
// its columns' weights in registers.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "gemm_common.h"
#include "kernels.h"

namespace ttamd {
namespace {

enum GateKind { GATE_NONE = 0, GATE_TOKEN = 1, GATE_CHANNEL = 2, GATE_FULL = 3 };

// 8 consecutive elements of bf16 or fp32.
__device__ __forceinline__ void load8(const void* p, int64_t i, bool f32, float* v) {
  if (f32) {
    const float4* q = (const float4*)((const float*)p + i);
    const float4 a = q[0], b = q[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    unpack8(*(const uint4*)((const bf16_t*)p + i), v);
  }
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
__device__ __forceinline__ float sigmoid_of(float g) { return 1.f / (1.f + expf(-g)); }

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
// Forward.  WAVE: one row per wave (4 per workgroup), else one per workgroup.
// ---------------------------------------------------------------------------
template <bool WAVE, int VPT, bool S32, bool COMBINE>
__global__ __launch_bounds__(WAVE ? 256 : 1024) void norm_forward_kernel(const NormArgs a) {
  __shared__ float slots[2][1][16];
  int phase = 0;
  const int tid = WAVE ? threadIdx.x & 63 : threadIdx.x;
  const int nt = WAVE ? 64 : blockDim.x;
  const int rows_wg = WAVE ? blockDim.x >> 6 : 1;
  const int D = a.D;
  int col[VPT];
  bool on[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    col[i] = 8 * (tid + i * nt);
    on[i] = col[i] < D;
  }
  // w_post * scale * act(channel gate), and w_pre, of vector i
  auto weights_u = [&](int i, float* w) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = 1.f;
    if (a.post && on[i]) load8(a.post, col[i], a.post32, w);
    float g[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = 1.f;
    if (a.gate_kind == GATE_CHANNEL && on[i]) {
      load8(a.gate, col[i], a.gate32, g);
      if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = sigmoid_of(g[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] *= a.scale * g[j];
  };
  auto weights_n = [&](int i, float* w) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = 0.f;
    if (a.pre && on[i]) load8(a.pre, col[i], a.pre32, w);
  };
  // a workgroup that holds few columns per thread keeps them, a wave reads
  // them again for every row (from L1: registers are worth more)
  constexpr int HOLD = WAVE ? 1 : VPT;
  float hold_u[HOLD][8], hold_n[HOLD][8];
  if constexpr (!WAVE) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      weights_u(i, hold_u[i]);
      weights_n(i, hold_n[i]);
    }
  }
  const float inv_d = 1.f / (float)D;
  const int64_t step = (int64_t)gridDim.x * rows_wg;
  for (int64_t t = (int64_t)blockIdx.x * rows_wg + (WAVE ? threadIdx.x >> 6 : 0); t < a.T; t += step) {
    float x[VPT][8];  // f, then u
    float r[VPT][8];
    const int64_t base = t * D;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = 0.f, r[i][j] = 0.f;
      if (on[i] && a.residual) load8(a.residual, base + col[i], S32, r[i]);
    }
    if constexpr (COMBINE) {
      for (int k = 0; k < a.K; ++k) {
        int64_t row = t * a.K + k;
        const float p = a.probs ? a.probs[row] : 1.f;
        if (a.inverse) row = min(max(a.inverse[row], 0), a.T * a.K - 1);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          if (on[i]) {
            float v[8];
            unpack8(load_stream((const uint4*)(a.rows + row * D + col[i])), v);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = fmaf(p, v[j], x[i][j]);
          }
        }
      }
    } else if (a.rows) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (on[i]) load8(a.rows, base + col[i], false, x[i]);
    }
    float gt = 1.f;
    if (a.gate_kind == GATE_TOKEN) {
      gt = load1(a.gate, t, a.gate32);
      if (a.sigmoid) gt = sigmoid_of(gt);
    }
    float gf[VPT][8];
    if (a.gate_kind == GATE_FULL) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (on[i]) load8(a.gate, base + col[i], a.gate32, gf[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) gf[i][j] = on[i] ? (a.sigmoid ? sigmoid_of(gf[i][j]) : gf[i][j]) : 0.f;
      }
    }
    float rf = 1.f;
    if (a.post) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] = fmaf(x[i][j], x[i][j], s[0]);
      if constexpr (WAVE) s[0] = wave64_sum(s[0]);
      else block_sums<1>(s, slots, phase);
      rf = 1.f / sqrtf(s[0] * inv_d + a.eps);
    }
    if (a.rows) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float w[8];
        if constexpr (WAVE) weights_u(i, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float g = gt * (WAVE ? w[j] : hold_u[WAVE ? 0 : i][j]);
          if (a.gate_kind == GATE_FULL) g *= gf[i][j];
          x[i][j] = r[i][j] + g * (x[i][j] * rf);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = r[i][j];
    }
    if (a.u) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (on[i]) store8(a.u, base + col[i], S32, x[i]);
    }
    float ru = 1.f;
    if (a.pre) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] = on[i] ? fmaf(x[i][j], x[i][j], s[0]) : s[0];
      if constexpr (WAVE) s[0] = wave64_sum(s[0]);
      else block_sums<1>(s, slots, phase);
      ru = 1.f / sqrtf(s[0] * inv_d + a.eps);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (on[i]) {
          float v[8], w[8];
          if constexpr (WAVE) weights_n(i, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = x[i][j] * ru * (WAVE ? w[j] : hold_n[WAVE ? 0 : i][j]);
          store8(a.n, base + col[i], false, v);
        }
      }
    }
    if (a.rstd && tid == 0) {
      a.rstd[t] = rf;
      a.rstd[a.T + t] = ru;
    }
  }
}

// ---------------------------------------------------------------------------
// Backward.  u is recomputed from the branch, the residual and the saved
// r_f, so the gradient is of exactly what the forward computed:
//   q = dn * w_pre;       dU = du + r_u (q - u r_u^2 mean(q u))
//   dresidual = dU;       dw_pre = sum_t dn u r_u
//   dp = scale a dU;      dgate = scale dU p act'   (summed over what it was broadcast)
//   q2 = dp * w_post;     df = r_f (q2 - f r_f^2 mean(q2 f));  dw_post = sum_t dp f r_f
// One workgroup per row at a time; the column sums of its rows stay in
// registers and leave once per workgroup as partial sums, which a second
// launch adds in workgroup order (no atomics: the same bits every time).
// ---------------------------------------------------------------------------
template <int VPT, bool S32>
__global__ __launch_bounds__(512) void norm_backward_kernel(const NormBwdArgs a) {
  __shared__ float slots1[2][1][16], slots2[2][2][16];
  int ph1 = 0, ph2 = 0;
  const NormArgs& f = a.fwd;
  const int tid = threadIdx.x, nt = blockDim.x, D = f.D;
  int col[VPT];
  bool on[VPT];
  float wpost[VPT][8], wpre[VPT][8], gch[VPT][8];
  float s_post[VPT][8], s_pre[VPT][8], s_gate[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    col[i] = 8 * (tid + i * nt);
    on[i] = col[i] < D;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      wpost[i][j] = 1.f, wpre[i][j] = 0.f, gch[i][j] = 1.f;
      s_post[i][j] = s_pre[i][j] = s_gate[i][j] = 0.f;
    }
    if (on[i]) {
      if (f.post) load8(f.post, col[i], f.post32, wpost[i]);
      if (f.pre) load8(f.pre, col[i], f.pre32, wpre[i]);
      if (f.gate_kind == GATE_CHANNEL) load8(f.gate, col[i], f.gate32, gch[i]);
    }
  }
  const float inv_d = 1.f / (float)D;
  for (int64_t t = blockIdx.x; t < f.T; t += gridDim.x) {
    const int64_t base = t * D;
    float x[VPT][8], u[VPT][8], g[VPT][8], dn[VPT][8];  // g: du, then dU
    float act[VPT][8], dact[VPT][8];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = u[i][j] = g[i][j] = dn[i][j] = 0.f;
      if (on[i]) {
        if (f.rows) load8(f.rows, base + col[i], false, x[i]);
        if (f.residual) load8(f.residual, base + col[i], S32, u[i]);
        if (a.du) load8(a.du, base + col[i], S32, g[i]);
        if (a.dn) load8(a.dn, base + col[i], false, dn[i]);
      }
    }
    const float rf = f.rstd[t], ru = f.rstd[f.T + t];
    // act(gate) and its derivative
    float gt = 1.f;
    if (f.gate_kind == GATE_TOKEN) gt = load1(f.gate, t, f.gate32);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float raw[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) raw[j] = f.gate_kind == GATE_TOKEN ? gt : gch[i][j];
      if (f.gate_kind == GATE_FULL && on[i]) load8(f.gate, base + col[i], f.gate32, raw);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        act[i][j] = raw[j], dact[i][j] = 1.f;
        if (f.sigmoid && f.gate_kind != GATE_NONE) {
          const float s = sigmoid_of(raw[j]);
          act[i][j] = s, dact[i][j] = s * (1.f - s);
        }
      }
    }
    if (f.rows) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) u[i][j] += f.scale * act[i][j] * (x[i][j] * rf * wpost[i][j]);
    }
    if (f.pre) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] = fmaf(dn[i][j] * wpre[i][j], u[i][j], s[0]);
      block_sums<1>(s, slots1, ph1);
      const float c = s[0] * inv_d * ru * ru;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          s_pre[i][j] = fmaf(dn[i][j], u[i][j] * ru, s_pre[i][j]);
          g[i][j] += ru * (dn[i][j] * wpre[i][j] - u[i][j] * c);
        }
    }
    if (a.dresidual) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (on[i]) store8(a.dresidual, base + col[i], S32, g[i]);
    }
    if (!f.rows) continue;  // uniform
    float s[2] = {0.f, 0.f};  // sum of q2 f, sum of dgate
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float dg[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float fh = x[i][j] * rf;
        dg[j] = f.scale * g[i][j] * (fh * wpost[i][j]) * dact[i][j];
        const float dp = f.scale * act[i][j] * g[i][j];
        s_post[i][j] = fmaf(dp, fh, s_post[i][j]);
        s_gate[i][j] += dg[j];
        s[1] += dg[j];
        g[i][j] = dp * wpost[i][j];
        s[0] = fmaf(g[i][j], x[i][j], s[0]);
      }
      if (f.gate_kind == GATE_FULL && a.dgate && on[i]) store8(a.dgate, base + col[i], f.gate32, dg);
    }
    if (f.post || f.gate_kind == GATE_TOKEN) block_sums<2>(s, slots2, ph2);
    const float c = f.post ? s[0] * inv_d * rf * rf : 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (on[i]) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = rf * (g[i][j] - x[i][j] * c);
        if (a.dbranch) store8(a.dbranch, base + col[i], false, v);
      }
    }
    if (f.gate_kind == GATE_TOKEN && a.dgate && tid == 0) {
      if (f.gate32) ((float*)a.dgate)[t] = s[1];
      else ((bf16_t*)a.dgate)[t] = (bf16_t)f32_to_bf16(s[1]);
    }
  }
  // partial sums of this workgroup's rows: [3][grid][D], unused ones skipped
  const int64_t plane = (int64_t)gridDim.x * D;
  float* part = a.part + (int64_t)blockIdx.x * D;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (on[i]) {
      if (a.dpost) store8(part, col[i], true, s_post[i]);
      if (a.dpre) store8(part + plane, col[i], true, s_pre[i]);
      if (a.dgate && f.gate_kind == GATE_CHANNEL) store8(part + 2 * plane, col[i], true, s_gate[i]);
    }
  }
}

// out[c] = sum of the n partial rows of column c, in order: 16 runs of rows
// side by side, then the runs.  blockIdx.y: which of the three sums.
struct ColumnSumArgs {
  const float* part;  // [3][n][D]
  int n, D;
  void* out[3];
  int f32[3];
};
__global__ __launch_bounds__(256) void column_sum_kernel(const ColumnSumArgs a) {
  __shared__ float4 sh[16][16];
  const int which = blockIdx.y;
  void* out = a.out[which];
  if (!out) return;
  const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4;
  const int c = (blockIdx.x * 16 + cx) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < a.D) {
    const float* p = a.part + (int64_t)which * a.n * a.D + c;
    const int per = (a.n + 15) / 16, r1 = min((ry + 1) * per, a.n);
    for (int r = ry * per; r < r1; ++r) {
      const float4 v = *(const float4*)(p + (int64_t)r * a.D);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  sh[ry][cx] = s;
  __syncthreads();
  if (ry == 0 && c < a.D) {
    for (int r = 1; r < 16; ++r) {
      const float4 v = sh[r][cx];
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    if (a.f32[which])
      *(float4*)((float*)out + c) = s;
    else
      *(uint2*)((bf16_t*)out + c) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
  }
}

int round64(int v) { return (v + 63) & ~63; }

template <bool S32, bool COMBINE>
hipError_t go_forward(const NormArgs& a, hipStream_t stream) {
  const int nvec = a.D / 8;
  const int64_t cap = 16LL * num_cus();
  if (nvec <= 256 && a.T > 8 * num_cus()) {
    const dim3 grid((unsigned)std::min<int64_t>((a.T + 3) / 4, cap));
    if (nvec <= 64) return launch_k(false, norm_forward_kernel<true, 1, S32, COMBINE>, grid, dim3(256), 0, stream, a);
    if (nvec <= 128) return launch_k(false, norm_forward_kernel<true, 2, S32, COMBINE>, grid, dim3(256), 0, stream, a);
    return launch_k(false, norm_forward_kernel<true, 4, S32, COMBINE>, grid, dim3(256), 0, stream, a);
  }
  const dim3 grid((unsigned)std::min<int64_t>(a.T, cap));
  return launch_k(false, norm_forward_kernel<false, 1, S32, COMBINE>, grid, dim3(round64(nvec)), 0, stream, a);
}

// Workgroups of the backward: enough to fill the chip, few enough that their
// partial sums stay small beside the rows.
int backward_groups(int64_t T) { return (int)std::min<int64_t>(T, 4 * (int64_t)num_cus()); }

}  // namespace

hipError_t launch_norm_forward(const NormArgs& a, hipStream_t stream) {
  if (a.T == 0) return hipSuccess;
  const bool combine = a.rows && (a.K > 1 || a.inverse || a.probs);
  if (a.stream32) return combine ? go_forward<true, true>(a, stream) : go_forward<true, false>(a, stream);
  return combine ? go_forward<false, true>(a, stream) : go_forward<false, false>(a, stream);
}

size_t norm_backward_workspace_bytes(int64_t T, int64_t D) {
  return 3 * (size_t)backward_groups(T) * (size_t)D * sizeof(float);
}

hipError_t launch_norm_backward(const NormBwdArgs& b, hipStream_t stream) {
  const NormArgs& a = b.fwd;
  if (a.T == 0) return hipSuccess;
  const int nvec = a.D / 8, groups = backward_groups(a.T);
  auto go = [&](auto vpt) {
    constexpr int VPT = decltype(vpt)::value;
    const dim3 block(round64((nvec + VPT - 1) / VPT));
    if (a.stream32) return launch_k(false, norm_backward_kernel<VPT, true>, dim3(groups), block, 0, stream, b);
    return launch_k(false, norm_backward_kernel<VPT, false>, dim3(groups), block, 0, stream, b);
  };
  hipError_t err = nvec <= 512 ? go(std::integral_constant<int, 1>{}) : go(std::integral_constant<int, 2>{});
  const bool channel = b.dgate && a.gate_kind == GATE_CHANNEL;
  if (err != hipSuccess || !(b.dpost || b.dpre || channel)) return err;
  ColumnSumArgs c = {};
  c.part = b.part;
  c.n = groups;
  c.D = a.D;
  c.out[0] = b.dpost, c.out[1] = b.dpre, c.out[2] = channel ? b.dgate : nullptr;
  c.f32[0] = a.post32, c.f32[1] = a.pre32, c.f32[2] = a.gate32;
  return launch_k(false, column_sum_kernel, dim3((a.D + 63) / 64, 3), dim3(256), 0, stream, c);
}

}  // namespace ttamd
