// 4-bit weights on MI355X (gfx950): e2m1 codes with one power-of-two scale for
// each 32 values along a row, packed once and read by the few-token kernels
// (decode.hip), and their restoration.
//
//   e    = the smallest integer with max |v| <= 6 * 2^e over the 32 values, at
//          least -126 and at most 125
//   code = e2m1(v * 2^-e): 0, 0.5, 1, 1.5, 2, 3, 4 or 6 and a sign, nearest,
//          ties to the even code (e = 125: at most 6, since 8 * 2^125 is past
//          bf16's range)
//   exponent byte = e + 127, or 255 where one of the 32 is a NaN or infinite:
//          the whole group is then NaN
//   value = code * 2^e, exact in bf16
//
// Layout: tiles of 16 rows and 128 columns, 1 KB, place l (0..63) of a tile holding
// the 32 columns 32 (l / 16) .. + 31 of row l % 16 in 16 bytes, low half byte
// first.  A wave's load of a tile is then one contiguous KB, and what it gets is
// what v_mfma_f32_16x16x32_bf16 wants: lane l's eight values of step j are bytes
// 4 j .. 4 j + 3 of its 16, all of one group, so that one conversion
// (v_cvt_scalef32_pk_bf16_fp4) takes two codes and their scale to two bf16.
// Exponents: [row tile][ceil(tiles along K / 4)][64 places][4 tiles], a dword per
// lane for four tiles.  Rows past N and columns past K hold zeros.
//
// Memory-bound: 2 (bf16) bytes in, 17/32 out, and back.
#include <algorithm>

#include "common.h"
#include "fp4.h"
#include "gemm_common.h"
#include "kernels.h"

namespace ttamd {
namespace {

// The exponent byte of 32 values whose largest finite |v| has these fp32 bits:
// |v| = 1.m * 2^(E - 127), 6 = 1.5 * 2^2.
__device__ __forceinline__ int exponent_byte(uint32_t bits) {
  const int e = (int)(bits >> 23) - 2 + ((bits & 0x7fffffu) > 0x400000u ? 1 : 0);
  return min(max(e, 127 - 126), 127 + 125);
}

// One wave per 16 rows and four tiles along K.
template <bool F32>
__global__ __launch_bounds__(256) void pack_fp4_kernel(const void* __restrict__ in, int N, int K, int NB, int C, int C4,
                                                       int64_t total, uint4* __restrict__ codes,
                                                       uint32_t* __restrict__ exps) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // (matrix, row tile, tile group)
  if (t >= total) return;
  const int l = threadIdx.x & 63;
  const int g = (int)(t % C4);
  const int64_t eb = t / C4;  // (matrix, row tile)
  const int row = 16 * (int)(eb % NB) + (l & 15);
  const int64_t at = (eb / NB * N + row) * (int64_t)K;
  uint32_t bytes = 0;
  for (int j = 0; j < 4; ++j) {
    const int c = 4 * g + j, k = 128 * c + 32 * (l >> 4);
    if (c >= C) {
      bytes |= 127u << (8 * j);
      continue;
    }
    float f[32];
    if (row < N && k < K) {
      if constexpr (F32) {
        const float4* p = (const float4*)((const float*)in + at + k);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 v = p[i];
          f[4 * i] = v.x, f[4 * i + 1] = v.y, f[4 * i + 2] = v.z, f[4 * i + 3] = v.w;
        }
      } else {
        const uint4* p = (const uint4*)((const bf16_t*)in + at + k);
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack8(p[i], f + 8 * i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] = 0.f;
    }
    uint32_t most = 0;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const uint32_t b = __float_as_uint(f[i]) & 0x7fffffffu;
      odd |= b >= 0x7f800000u;
      most = max(most, b);
    }
    const int e = odd ? 255 : exponent_byte(most);
    const float scale = __uint_as_float((uint32_t)(odd ? 127 : e) << 23);
    uint32_t q[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      q[d] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[8 * d], f[8 * d + 1], scale, 0);
      q[d] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q[d], f[8 * d + 2], f[8 * d + 3], scale, 1);
      q[d] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q[d], f[8 * d + 4], f[8 * d + 5], scale, 2);
      q[d] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q[d], f[8 * d + 6], f[8 * d + 7], scale, 3);
      if (odd) q[d] = 0;
    }
    codes[(eb * C + c) * 64 + l] = make_uint4(q[0], q[1], q[2], q[3]);
    bytes |= (uint32_t)e << (8 * j);
  }
  exps[t * 64 + l] = bytes;
}

__global__ __launch_bounds__(256) void unpack_fp4_kernel(const uint4* __restrict__ codes,
                                                         const uint32_t* __restrict__ exps, int N, int K, int NB, int C,
                                                         int C4, int64_t total, bf16_t* __restrict__ out) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= total) return;
  const int l = threadIdx.x & 63;
  const int g = (int)(t % C4);
  const int64_t eb = t / C4;
  const int row = 16 * (int)(eb % NB) + (l & 15);
  if (row >= N) return;
  const int64_t at = (eb / NB * N + row) * (int64_t)K;
  const uint32_t bytes = exps[t * 64 + l];
  for (int j = 0; j < 4; ++j) {
    const int c = 4 * g + j, k = 128 * c + 32 * (l >> 4);
    if (c >= C || k >= K) break;
    const uint4 q = codes[(eb * C + c) * 64 + l];
    const float scale = fp4_scale(bytes, j);
    uint4* p = (uint4*)(out + at + k);
    p[0] = fp4_bits(q.x, scale), p[1] = fp4_bits(q.y, scale);
    p[2] = fp4_bits(q.z, scale), p[3] = fp4_bits(q.w, scale);
  }
}

}  // namespace

hipError_t launch_pack_fp4(const void* in, bool f32, int64_t E, int N, int K, void* codes, void* exps,
                           hipStream_t stream) {
  const int NB = (N + 15) / 16, C = (K + 127) / 128, C4 = (C + 3) / 4;
  const int64_t total = E * NB * C4;
  if (total == 0) return hipSuccess;
  const dim3 grid((unsigned)((total + 3) / 4));
  auto kernel = f32 ? pack_fp4_kernel<true> : pack_fp4_kernel<false>;
  return launch_k(false, kernel, grid, dim3(256), 0, stream, in, N, K, NB, C, C4, total, (uint4*)codes,
                  (uint32_t*)exps);
}

hipError_t launch_unpack_fp4(const void* codes, const void* exps, int64_t E, int N, int K, void* out,
                             hipStream_t stream) {
  const int NB = (N + 15) / 16, C = (K + 127) / 128, C4 = (C + 3) / 4;
  const int64_t total = E * NB * C4;
  if (total == 0) return hipSuccess;
  return launch_k(false, unpack_fp4_kernel, dim3((unsigned)((total + 3) / 4)), dim3(256), 0, stream,
                  (const uint4*)codes, (const uint32_t*)exps, N, K, NB, C, C4, total, (bf16_t*)out);
}

}  // namespace ttamd
