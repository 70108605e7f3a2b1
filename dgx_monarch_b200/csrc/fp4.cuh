// What the microscaled 4-bit kernels share: the formats, the layout of a
// packed tensor and its decoding.
//
// A (rows, cols) tensor is held as
//   values  rows of fp4_pitch(cols) bytes, two e2m1 codes a byte (the even
//           column in the low bits), zero past the last column;
//   scales  one byte for each row and block of columns, in tiles of 128 rows x
//           4 blocks, 512 bytes each, row tiles outermost: the byte of row r and block b
//           of a tile is at (r % 32) * 16 + (r / 32) * 4 + b -- the order in
//           which tcgen05.cp spreads it over tensor memory.  Zero past the
//           last block; rows past the last one are not written;
//   scale   nvfp4: one fp32 for the tensor.
// nvfp4: blocks of 16, e4m3 scales s, value = code s scale.
// mxfp4: blocks of 32, e8m0 scales (2^(byte - 127)), value = code s.
// A NaN scale byte (0x7F, 0xFF) makes its block NaN.
#pragma once

#include "common.h"
#include "ptx.cuh"

namespace dgxm {

__host__ __device__ constexpr int fp4_block(int format) { return format == DGXM_FP4_NVFP4 ? 16 : 32; }
__host__ __device__ constexpr int64_t fp4_pitch(int64_t cols) { return (cols + 31) / 32 * 16; }
__host__ __device__ constexpr int64_t fp4_groups(int64_t cols, int format) {
  return (cols + 4 * fp4_block(format) - 1) / (4 * fp4_block(format));
}
__host__ __device__ constexpr int64_t fp4_scale_at(int64_t row, int64_t block, int64_t groups) {
  return ((row >> 7) * groups + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// The float that a scale byte stands for.
template <int FORMAT>
__device__ __forceinline__ float fp4_scale_value(uint32_t byte) {
  if constexpr (FORMAT == DGXM_FP4_NVFP4)
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
  else  // 2^-127 is the one subnormal
    return byte == 0 ? __uint_as_float(1u << 22) : __uint_as_float(byte == 255 ? 0x7FC00000u : byte << 23);
}

// Eight e2m1 codes (low bits first) of a word as halves; every one is exact.
__device__ __forceinline__ void fp4_decode8(uint32_t codes, __half2 (&out)[4]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = *reinterpret_cast<__half2*>(&h[i]);
}

// Eight floats to e2m1 codes, nearest, ties to the even code, saturating.
__device__ __forceinline__ uint32_t fp4_encode8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}\n"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// A scale that a caller gives in device memory, in one of three types.
__device__ __forceinline__ float fp4_read_scale(const void* p, int dtype) {
  if (dtype == DGXM_DTYPE_BF16) return __bfloat162float(*static_cast<const __nv_bfloat16*>(p));
  if (dtype == DGXM_DTYPE_F16) return __half2float(*static_cast<const __half*>(p));
  return *static_cast<const float*>(p);
}

}  // namespace dgxm
