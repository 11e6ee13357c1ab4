// Microscaled 4-bit operands: layout, decoding and the rounding of one block.
//
// Values are e2m1 (sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6) times a
// block scale: MXFP4 blocks of 32 with an e8m0 scale (a power of two, byte - 127), NVFP4 blocks
// of 16 with an e4m3 scale and a tensor scale that is a power of two.
//
// Layout.  codes: [rows][P / 2] bytes, P = n rounded up to 256, element 2j of a row in the low
// half of byte j.  scales: tiles of 128 rows x 4 blocks, 512 bytes each, [row tile][block
// group][32][4][4]: byte 16 r + 4 j + k of a tile is row 32 j + r, block k.  That is the order in
// which the block-scaled MMA wants a tile's scales in tensor memory (lane r, column j, byte k), so
// they go there by plain copies.  Codes and scales past n are zero; the scale bytes of rows past
// the last are never used.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "mx4_kernels.h"

namespace cpk {

template <int FMT> __host__ __device__ constexpr int mx_block() { return FMT == kMXFP4 ? 32 : 16; }
template <int FMT> __host__ __device__ constexpr int mx_nan_scale() { return FMT == kMXFP4 ? 0xFF : 0x7F; }

// Byte offset of (row, block) in the scale tiles; groups = P / (4 * block size).
__host__ __device__ __forceinline__ int64_t mx_scale_offset(int64_t row, int64_t blk, int64_t groups) {
  return ((row >> 7) * groups + (blk >> 2)) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (blk & 3);
}

// e8m0 byte -> 2^(byte - 127) (255: NaN).
__device__ __forceinline__ float e8m0_value(uint32_t b) {
  return b == 255 ? __int_as_float(0x7FC00000) : __int_as_float(b ? b << 23 : 0x00400000);
}
// e4m3 byte (sign ignored) -> value; 0x7F: NaN.
__device__ __forceinline__ float e4m3_value(uint32_t b) {
  uint32_t h;
  asm("{\n\t.reg .b16 s;\n\tcvt.u16.u32 s, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, s;\n\t}" : "=r"(h) : "r"(b & 0x7F));
  return __half2float(__ushort_as_half((unsigned short)(h & 0xFFFF)));
}
template <int FMT> __device__ __forceinline__ float mx_scale_value(uint32_t b) {
  return FMT == kMXFP4 ? e8m0_value(b) : e4m3_value(b);
}
// Two codes (low half first) -> their values.
__device__ __forceinline__ float2 e2m1x2_value(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 c, z;\n\t.reg .b16 s;\n\tcvt.u16.u32 s, %1;\n\tmov.b16 {c, z}, s;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, c;\n\t}"
      : "=r"(h)
      : "r"(byte & 0xFF));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}
// Eight values -> eight codes, round to nearest even, saturating at 6.
__device__ __forceinline__ uint32_t e2m1x8(const float (&q)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return r;
}

// Largest of a block's magnitudes, as bits (a NaN or infinity is >= 0x7F800000 and wins); lanes
// of a block hold 8 values each: 4 lanes for MXFP4, 2 for NVFP4.
template <int FMT> __device__ __forceinline__ uint32_t mx_block_max(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  if (FMT == kMXFP4) m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  return m;
}

// Scale byte of a block whose largest magnitude has the bits m.
//   MXFP4: floor(log2 max) - 2, the exponent at which the maximum lies in [4, 8).
//   NVFP4: the e4m3 nearest to max / 6.  The quotient is rounded to odd first (truncated, with a
//   last bit that says whether anything was cut), so the second rounding is the only one that
//   counts; max arrives already divided by the tensor scale.
template <int FMT> __device__ __forceinline__ int mx_first_scale(uint32_t m) {
  if (m >= 0x7F800000u) return mx_nan_scale<FMT>();
  if (FMT == kMXFP4) return max((int)(m >> 23) - 2, 0);
  const float a = __uint_as_float(m);
  float q = __fdiv_rz(a, 6.0f);
  if (__fmaf_rn(q, 6.0f, -a) != 0.0f) q = __uint_as_float(__float_as_uint(q) | 1u);
  uint32_t r;
  asm("{\n\t.reg .b16 s;\n\tcvt.rn.satfinite.e4m3x2.f32 s, %1, %1;\n\tcvt.u32.u16 %0, s;\n\t}" : "=r"(r) : "f"(q));
  return (int)(r & 0x7F);
}

// Codes of eight values against a block's scale.
//   MXFP4: v / 2^e is exact, so the conversion's rounding is the only one.
//   NVFP4: v / s is not.  t is the multiple of 1/4 nearest to the approximate quotient, and every
//   border between two e2m1 values is such a multiple.  t s is exact (t has at most 5 bits where
//   a border can lie, s has 4) and r = v - t s has the right sign, so t + 1.9 r / s, which stays
//   within a quarter of t, is on the side of t that v is on, and is t itself on a tie.
template <int FMT> __device__ __forceinline__ uint32_t mx_codes(const float (&v)[8], int byte) {
  float q[8];
  if (FMT == kMXFP4) {
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);   // byte <= 253: a normal power of two
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = __fmul_rn(v[i], inv);
  } else {
    const float s = e4m3_value(byte);
    const float inv = s > 0.0f ? __frcp_rn(s) : 0.0f;
    const float slope = 1.9f * inv;
    constexpr float kQuarter = 3145728.0f;   // 1.5 * 2^21: adding it rounds to a multiple of 1/4
#pragma unroll
    for (int i = 0; i < 8; i++) {
      // the clamp keeps the magic addition in range; past 8 every value is 6
      const float a = fminf(fmaxf(__fmul_rn(v[i], inv), -64.0f), 64.0f);
      const float t = __fsub_rn(__fadd_rn(a, kQuarter), kQuarter);
      const float r = __fmaf_rn(-t, s, v[i]);
      // +0 for t keeps the sign of v on values that round to zero; it does not matter to any sum
      q[i] = __fmaf_rn(r, slope, t);
    }
  }
  return e2m1x8(q);
}

}  // namespace cpk
