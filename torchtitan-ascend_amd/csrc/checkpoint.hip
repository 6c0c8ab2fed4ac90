// Activation checkpoints in 8 bits on MI355X (gfx950): bf16 rows stored as
// e4m3 codes with one power-of-two scale per row and 128 columns, and their
// restoration (whole, or rows gathered in routing order).
//
//   e    = the smallest integer with max |v| <= 448 * 2^e over the block's
//          finite values, at least -118 and at most 120
//   code = e4m3fn(v * 2^-e), nearest, ties to even;  NaN and inf: 0x7f (NaN)
//          (e = 120: at most 240, since 256 * 2^120 is past bf16's range)
//   exponent byte = e + 127
//   value = code * 2^e
//
// A power of two (not absmax / 448) makes the value exact in bf16: e4m3 has
// four significant bits, bf16 eight, so a restored row goes to the matrix
// cores, or an epilogue rebuilds it, without a second rounding.  It costs at
// most half a binade of range, none of the code's relative precision.  Blocks
// below 448 * 2^-118 lose range at the bottom: their least code is 2^-127, a
// subnormal number of bf16 and fp32 (kept by every step here), where the scale
// of a lower exponent would lead out of bf16.
//
// Memory-bound: 2 bytes in, 1 + 1/128 out (back: the reverse).  16 lanes share
// a block, 8 columns (16 bytes) each; the maximum is an integer maximum of the
// bf16 bits (ordered as the values are), the exponent comes from its bits, and
// v_cvt_pk_fp8_f32 rounds.  Measured (65536 rows of 1536): pack 54 us, unpack
// 48 us, 5.6 and 6.3 TB/s; 1003 rows of 1544 4.2 and 3.4 us, a launch each.
#include <algorithm>

#include "common.h"
#include "gemm_common.h"
#include "kernels.h"

namespace ttamd {
namespace {

constexpr int kUnroll = 4;  // blocks per 16 lanes at a time: loads in flight

__device__ __forceinline__ int row16_imax(int v) {
  v = max(v, dpp_i<kDppXor1>(v));
  v = max(v, dpp_i<kDppXor2>(v));
  v = max(v, dpp_i<kDppHalfMirror>(v));
  return max(v, dpp_i<kDppMirror>(v));
}

// Exponent byte of a block whose largest finite |v| has these bf16 bits.
__device__ __forceinline__ int exponent_byte(int bits) {
  // |v| = 1.m * 2^(E - 127); 448 = 1.75 * 2^8: e = E - 127 - 8, one more above 1.75
  return min(max((bits >> 7) - 8 + ((bits & 0x7f) > 0x60 ? 1 : 0), 127 - 118), 127 + 120);
}

// Block `blk` of the tensor (row-major over [R, nb]): 128 columns of a row.
// EXACT: C % 128 == 0, blocks follow one another in memory.
template <bool EXACT>
__global__ __launch_bounds__(256) void pack_rows_kernel(const uint4* __restrict__ in, uint32_t nblocks, uint32_t nb,
                                                        uint32_t cv, uint2* __restrict__ codes,
                                                        uint8_t* __restrict__ exps) {
  const uint32_t l16 = threadIdx.x & 15;
  const uint32_t stride = gridDim.x * 16;  // indices stay below 2^31: the caller's
  for (uint32_t b0 = blockIdx.x * 16 + (threadIdx.x >> 4); b0 < nblocks; b0 += kUnroll * stride) {
    uint4 v[kUnroll];
    uint32_t at[kUnroll];
    bool on[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const uint32_t blk = b0 + i * stride;
      on[i] = blk < nblocks;
      if constexpr (EXACT) {
        at[i] = blk * 16 + l16;
      } else {
        const uint32_t row = blk / nb, c = (blk - row * nb) * 16 + l16;
        on[i] = on[i] && c < cv;
        at[i] = row * cv + c;
      }
      v[i] = on[i] ? load_stream(in + at[i]) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      int most = 0;
      bool odd = false;  // a NaN or inf
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int lo = (int)(w[d] & 0x7fffu), hi = (int)((w[d] >> 16) & 0x7fffu);
        odd |= lo >= 0x7f80 || hi >= 0x7f80;
        most = max(most, max(lo < 0x7f80 ? lo : 0, hi < 0x7f80 ? hi : 0));
      }
      const int e = exponent_byte(row16_imax(most));
      const float inv = __uint_as_float((uint32_t)(254 - e) << 23);  // 2^-(e - 127)
      float f[8];
      unpack8(v[i], f);
      // 2^128 would not be a bf16 number: the topmost block's codes end at 240
      if (__builtin_amdgcn_ballot_w64(e == 127 + 120)) {
        const float top = e == 127 + 120 ? __uint_as_float((127u + 120 + 7) << 23) * 1.875f : INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = fminf(fmaxf(f[j], -top), top);
      }
      int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * inv, f[1] * inv, 0, false);
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * inv, f[3] * inv, lo, true);
      int hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * inv, f[5] * inv, 0, false);
      hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] * inv, f[7] * inv, hi, true);
      if (__builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (((j & 1 ? w[j >> 1] >> 16 : w[j >> 1]) & 0x7fffu) >= 0x7f80u) {
            int& q = j < 4 ? lo : hi;
            q = (q & ~(0xff << (8 * (j & 3)))) | (0x7f << (8 * (j & 3)));
          }
        }
      }
      if (on[i]) codes[at[i]] = make_uint2((uint32_t)lo, (uint32_t)hi);
      if (l16 == 0 && b0 + i * stride < nblocks) exps[b0 + i * stride] = (uint8_t)e;
    }
  }
}

// 8 columns per lane and step.  With n_ids > 0 the grid also resolves the
// routed rows' ids, and pads them by 64 for the GEMM that reads them a stage
// at a time.
template <bool SCALE>
__global__ __launch_bounds__(256) void unpack_rows_kernel(const uint2* __restrict__ codes,
                                                          const uint8_t* __restrict__ exps, int n_src,
                                                          const int* __restrict__ src_index, int src_div,
                                                          const float* __restrict__ row_scale, uint32_t total,
                                                          uint32_t cv, uint32_t nb, uint4* __restrict__ out,
                                                          const int* __restrict__ ids_index, int* __restrict__ ids_out,
                                                          int n_ids) {
  const uint32_t threads = gridDim.x * 256, t0 = blockIdx.x * 256 + threadIdx.x;
  if (n_ids > 0) {
    for (uint32_t i = t0; i < (uint32_t)n_ids + 64; i += threads)
      ids_out[i] = i < (uint32_t)n_ids ? min(max(ids_index[i] / src_div, 0), n_src - 1) : 0;
  }
  for (uint32_t i0 = t0; i0 < total; i0 += kUnroll * threads) {
    uint2 q[kUnroll];
    int e[kUnroll];
    float mul[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const uint32_t at = i0 + i * threads;
      if (at >= total) continue;
      const uint32_t row = at / cv, c = at - row * cv;
      int64_t src = row;
      if (src_index) src = min(max(src_index[row] / src_div, 0), n_src - 1);
      q[i] = codes[src * cv + c];
      e[i] = exps[src * nb + (c >> 4)];
      mul[i] = SCALE ? row_scale[row] : 1.f;
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const uint32_t at = i0 + i * threads;
      if (at >= total) continue;
      const float s = __uint_as_float((uint32_t)e[i] << 23);
      float f[8];
      unpack_e4m3x4(q[i].x, s, f);
      unpack_e4m3x4(q[i].y, s, f + 4);
      if constexpr (SCALE) {
        // the stored bf16 value times the score, rounded once: a dispatched row
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= mul[i];
      }
      out[at] = pack8(f);
    }
  }
}

}  // namespace

hipError_t launch_pack_rows(const void* in, int64_t R, int C, void* codes, void* exps, hipStream_t stream) {
  const int nb = (C + 127) / 128;
  const int64_t nblocks = R * nb;
  if (nblocks == 0) return hipSuccess;
  const int64_t groups = (nblocks + 16 * kUnroll - 1) / (16 * kUnroll);
  const dim3 grid((unsigned)std::min<int64_t>(groups, 32 * num_cus()));
  if (C % 128 == 0)
    return launch_k(false, pack_rows_kernel<true>, grid, dim3(256), 0, stream, (const uint4*)in, (uint32_t)nblocks, nb,
                    C / 8, (uint2*)codes, (uint8_t*)exps);
  return launch_k(false, pack_rows_kernel<false>, grid, dim3(256), 0, stream, (const uint4*)in, (uint32_t)nblocks, nb,
                  C / 8, (uint2*)codes, (uint8_t*)exps);
}

hipError_t launch_unpack_rows(const void* codes, const void* exps, int n_src, const int* src_index, int src_div,
                              const float* row_scale, int64_t R, int C, void* out, const int* ids_index, int* ids_out,
                              int n_ids, hipStream_t stream) {
  const int64_t total = R * (C / 8);
  if (!ids_index || !ids_out) n_ids = 0;
  if (total == 0 && n_ids == 0) return hipSuccess;
  const int64_t work = std::max<int64_t>((total + kUnroll - 1) / kUnroll, n_ids);
  const dim3 grid((unsigned)std::min<int64_t>((work + 255) / 256, 32 * num_cus()));
  const int nb = (C + 127) / 128;
  if (row_scale)
    return launch_k(false, unpack_rows_kernel<true>, grid, dim3(256), 0, stream, (const uint2*)codes,
                    (const uint8_t*)exps, n_src, src_index, src_div, row_scale, (uint32_t)total, C / 8, nb,
                    (uint4*)out, ids_index, ids_out, n_ids);
  return launch_k(false, unpack_rows_kernel<false>, grid, dim3(256), 0, stream, (const uint2*)codes,
                  (const uint8_t*)exps, n_src, src_index, src_div, row_scale, (uint32_t)total, C / 8, nb, (uint4*)out,
                  ids_index, ids_out, n_ids);
}

}  // namespace ttamd
