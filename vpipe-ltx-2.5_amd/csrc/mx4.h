// Device helpers of the microscaled 4-bit formats (E2M1 codes, an E8M0 exponent for
// each block of 32), and the launchers that their C ABI layer (capi_mx4.cpp) calls.
#pragma once

#include "common.h"

namespace ltx25 {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// Where codes and scales lie (include/ltx25_mx4.h). Codes: tiles of 16 rows x 128 values,
// 1 KB; lane l of a wave reads the tile's 16 bytes l, block l / 16 of row l % 16. Scales:
// tiles of 16 rows x 16 blocks, 256 bytes; lane l reads dword l, its four blocks' for the
// four matrix instructions that span the tile's 512 values. An instruction takes a lane's
// block and scale from the same lane, so that no byte changes lanes; and four lanes side by
// side read 64 bytes: from rows of K / 2 bytes the same fragment takes the address unit four
// times as long (a wave's rows straight to registers: 91% of the time, matrix cores 36%).
constexpr int kMx4CodeTile = 1024;
constexpr int kMx4Tile = 256;
__host__ __device__ inline int mx4_slices(int K) { return (K + 127) / 128; }
__host__ __device__ inline int mx4_spans(int K) { return (K + 511) / 512; }
__host__ __device__ inline size_t mx4_code_bytes(long rows, int K)
{
  return (size_t)((rows + 15) / 16) * mx4_slices(K) * kMx4CodeTile;
}
__host__ __device__ inline size_t mx4_scale_bytes(long rows, int K)
{
  return (size_t)((rows + 15) / 16) * mx4_spans(K) * kMx4Tile;
}
// Within their tiles
__device__ __forceinline__ int mx4_code_at(int row, int block)
{
  return ((block & 3) * 16 + (row & 15)) * 16;
}
__device__ __forceinline__ int mx4_scale_at(int row, int block)
{
  return ((block & 3) * 16 + (row & 15)) * 4 + ((block >> 2) & 3);
}

// The exponent byte of a block whose largest magnitude has these bits (as f32):
// floor(log2) - 2 + 127, not below 0; 255 where it is no finite number.
__device__ __forceinline__ uint32_t mx4_scale(uint32_t top)
{
  const uint32_t e = top >> 23;
  return e == 255 ? 255u : (uint32_t)max((int)e - 2, 0);
}
// Eight values over 2^exponent to codes, the first in the low bits: to the nearest, ties to the
// even code, beyond 6 to 6 (the conversion's own rule). It divides by 2^exponent, of which its
// scale operand holds the bits: the exponent byte is f32's own, 0 for 2^-127 too.
__device__ __forceinline__ uint32_t mx4_codes(const float (&v)[8], float unit)
{
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], unit, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], unit, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], unit, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], unit, 3);
  return r;
}

// The larger of v over the lane's four (lanes 4 n .. 4 n + 3)
__device__ __forceinline__ uint32_t quad_max(uint32_t v)
{
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));   // 1 0 3 2
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));   // 2 3 0 1
  return v;
}

// A block of 32 held by four lanes, eight values each: its exponent byte and the
// lane's eight codes
__device__ __forceinline__ uint32_t mx4_code_quad(const float (&v)[8], uint32_t& scale)
{
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) { top = max(top, __float_as_uint(v[i]) & 0x7fffffffu); }
  scale = mx4_scale(quad_max(top));
  return scale == 255u ? 0u : mx4_codes(v, __uint_as_float(scale << 23));
}

// The same of bf16 values as they lie in memory
__device__ __forceinline__ uint32_t mx4_code_bf16_quad(uint4 raw, uint32_t& scale)
{
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  u16x2 top = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
  }
  scale = mx4_scale(quad_max((uint32_t)max((int)top[0], (int)top[1]) << 16));
  const float unit = __uint_as_float(scale << 23);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[0]), unit, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[1]), unit, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[2]), unit, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[3]), unit, 3);
  return scale == 255u ? 0u : r;
}

// A matrix operand of a lane: 32 codes, in the low half of the instruction's register
// list (4-bit operands do not use the rest)
__device__ __forceinline__ i32x8 mx4_operand(i32x4 v)
{
  return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
}
constexpr int kMfmaFp4 = 4;   // the instruction's format number of E2M1

// ---- launchers --------------------------------------------------------------

// An operand: `rows` rows of K values
struct Mx4Args {
  uint8_t* codes = nullptr;
  uint8_t* scales = nullptr;
  int rows = 0, K = 0;
};
hipError_t launch_mx4_quantize(const void* x, bool wide, int64_t stride, const Mx4Args& q,
                               hipStream_t stream);
hipError_t launch_mx4_dequant(const Mx4Args& q, uint16_t* out, int64_t stride, hipStream_t stream);
hipError_t launch_mx4_pack(const uint8_t* codes, const uint8_t* scales, const Mx4Args& q,
                           hipStream_t stream);
hipError_t launch_mx4_unpack(const Mx4Args& q, uint8_t* codes, uint8_t* scales, hipStream_t stream);

// y = epilogue(x . w^T + bias). `xb` set: bf16 activations at xb_stride, coded on the
// way; x then says where their codes go where the plan codes them ahead.
struct Mx4Gemm {
  Mx4Args x, w;
  const uint16_t* xb = nullptr;
  int64_t xb_stride = 0;
  const void* bias = nullptr;
  int bias_type = kBiasNone;
  int epilogue = kEpiNone;
  uint16_t* y = nullptr;
};
// The kernel and tile of a product; a function of the sizes alone.
struct Mx4Plan {
  int tile = 0;
  bool codes_ahead = false;   // bf16 activations are coded by a launch ahead
};
// `bf16`: the activations come in bf16
Mx4Plan plan_mx4(int M, int K, int N, bool bf16);
hipError_t launch_mx4_gemm(const Mx4Gemm& g, const Mx4Plan& plan, hipStream_t stream);

}  // namespace ltx25
