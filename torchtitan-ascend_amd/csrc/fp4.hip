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
// lane for four tiles.  Codes past N or K are zeros; exponents there are those of a
// group of zeros, or 127 in tiles past K (never 255, whose NaN would reach the sums).
//
// Memory-bound: 2 (bf16) bytes in, 17/32 out, and back.  A wave takes 16 rows of 512
// columns through LDS (rows 16 bytes apart from a multiple of 256: no bank
// conflicts), so that memory sees a whole KB of a row at a time; a place's own 64
// bytes, four pieces of 16, ran at 3.3 TB/s for the restoration and 4.7 for packing.
// Measured (128 matrices of 1536 x 2048): pack 164 us, restore 175, 6.2 and 5.8 TB/s;
// one of 1000 x 1440 4.9 and 4.0 us, a launch each.  fp32 weights (4 bytes in) are read
// by places, not through LDS: 435 us, 4.2 TB/s.
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

constexpr int kRowStride = 1024 + 16;
constexpr int kWaveLds = 16 * kRowStride;

// Codes of a place's 32 values into q, its exponent byte returned.
__device__ __forceinline__ uint32_t pack_group(const float (&f)[32], uint4& q) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) most = max(most, __float_as_uint(f[i]) & 0x7fffffffu);
  const bool odd = most >= 0x7f800000u;  // a NaN or an infinity is the largest of all
  const int e = odd ? 255 : exponent_byte(most);
  const float scale = __uint_as_float((uint32_t)(odd ? 127 : e) << 23);
  uint32_t d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    d[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[8 * i], f[8 * i + 1], scale, 0);
    d[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d[i], f[8 * i + 2], f[8 * i + 3], scale, 1);
    d[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d[i], f[8 * i + 4], f[8 * i + 5], scale, 2);
    d[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d[i], f[8 * i + 6], f[8 * i + 7], scale, 3);
    if (odd) d[i] = 0;
  }
  q = make_uint4(d[0], d[1], d[2], d[3]);
  return (uint32_t)e;
}

// One wave per 16 rows and four tiles along K.
template <bool F32>
__global__ __launch_bounds__(256) void pack_fp4_kernel(const void* __restrict__ in, int N, int K, int NB, int C, int C4,
                                                       int64_t total, uint4* __restrict__ codes,
                                                       uint32_t* __restrict__ exps) {
  __shared__ __attribute__((aligned(16))) char smem[F32 ? 16 : 4 * kWaveLds];
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // (matrix, row tile, tile group)
  if (t >= total) return;
  const int l = threadIdx.x & 63;
  const int g = (int)(t % C4);
  const int64_t eb = t / C4;  // (matrix, row tile)
  const int r0 = 16 * (int)(eb % NB);
  const int64_t at = eb / NB * N * (int64_t)K;
  char* const rows = smem + (F32 ? 0 : (threadIdx.x >> 6) * kWaveLds);
  if constexpr (!F32) {
    const int k = 512 * g + 8 * l;
    uint4 v[16];
#pragma unroll
    for (int r = 0; r < 16; ++r)
      v[r] = r0 + r < N && k < K ? load_stream((const uint4*)((const bf16_t*)in + at + (int64_t)(r0 + r) * K + k))
                                 : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int r = 0; r < 16; ++r) *(uint4*)(rows + r * kRowStride + 16 * l) = v[r];
    lds_wait();
  }
  uint32_t bytes = 0;
  const int row = r0 + (l & 15);
#pragma unroll 1
  for (int j = 0; j < 4; ++j) {
    const int c = 4 * g + j, k = 128 * c + 32 * (l >> 4);
    if (c >= C) {
      bytes |= 127u << (8 * j);
      continue;
    }
    float f[32];
    if constexpr (F32) {
      const float4* p = (const float4*)((const float*)in + at + (int64_t)row * K + k);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 v = row < N && k < K ? p[i] : make_float4(0.f, 0.f, 0.f, 0.f);
        f[4 * i] = v.x, f[4 * i + 1] = v.y, f[4 * i + 2] = v.z, f[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        unpack8(*(const uint4*)(rows + (l & 15) * kRowStride + 256 * j + 64 * (l >> 4) + 16 * i), f + 8 * i);
    }
    uint4 q;
    bytes |= pack_group(f, q) << (8 * j);
    store_stream(codes + (eb * C + c) * 64 + l, q);
  }
  exps[t * 64 + l] = bytes;
}

__global__ __launch_bounds__(256) void unpack_fp4_kernel(const uint4* __restrict__ codes,
                                                         const uint32_t* __restrict__ exps, int N, int K, int NB, int C,
                                                         int C4, int64_t total, bf16_t* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) char smem[4 * kWaveLds];
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= total) return;
  const int l = threadIdx.x & 63;
  const int g = (int)(t % C4);
  const int64_t eb = t / C4;
  const int r0 = 16 * (int)(eb % NB);
  char* const rows = smem + (threadIdx.x >> 6) * kWaveLds;
  const uint32_t bytes = exps[t * 64 + l];
  uint4 q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    q[j] = 4 * g + j < C ? load_stream(codes + (eb * C + 4 * g + j) * 64 + l) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float scale = fp4_scale(bytes, j);
    uint4* p = (uint4*)(rows + (l & 15) * kRowStride + 256 * j + 64 * (l >> 4));
    p[0] = fp4_bits(q[j].x, scale), p[1] = fp4_bits(q[j].y, scale);
    p[2] = fp4_bits(q[j].z, scale), p[3] = fp4_bits(q[j].w, scale);
  }
  lds_wait();
  const int k = 512 * g + 8 * l;
  if (k >= K) return;
  bf16_t* const to = out + (eb / NB * N + r0) * (int64_t)K + k;
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (r0 + r < N) store_stream((uint4*)(to + (int64_t)r * K), *(const uint4*)(rows + r * kRowStride + 16 * l));
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
