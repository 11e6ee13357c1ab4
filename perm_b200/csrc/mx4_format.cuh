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
// the last are written as zeros and never used.
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
// Eight values (four pairs) -> eight codes, round to nearest even, saturating at 6.
__device__ __forceinline__ uint32_t e2m1x8(const float2* q) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(q[0].x), "f"(q[0].y), "f"(q[1].x), "f"(q[1].y), "f"(q[2].x), "f"(q[2].y), "f"(q[3].x), "f"(q[3].y));
  return r;
}

// Largest of a block's magnitudes, as bits (a NaN or infinity is >= 0x7F800000 and wins), from the
// largest of each of its LANES lanes.
template <int LANES> __device__ __forceinline__ uint32_t mx_block_max(uint32_t m) {
#pragma unroll
  for (int o = 1; o < LANES; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// Scale byte of a block whose largest magnitude has the bits m.
//   MXFP4: floor(log2 max) - 2, the exponent at which the maximum lies in [4, 8).
//   NVFP4: the e4m3 nearest to max / (6 tensor_scale).  t is the approximate quotient cut to nine
//   significant bits; the borders between e4m3 values have five.  r = a - 6 t has the right sign, and
//   t + 1.9 r / 6, which stays short of t's neighbours, is on the side of t that a / 6 is on (t itself if
//   they are equal), so the conversion's rounding is that of the exact quotient.
template <int FMT> __device__ __forceinline__ int mx_first_scale(uint32_t m, float inv_tensor_scale) {
  if (FMT == kMXFP4) return m >= 0x7F800000u ? mx_nan_scale<FMT>() : max((int)(m >> 23) - 2, 0);
  const float a = fminf(__fmul_rn(__uint_as_float(m), inv_tensor_scale), 3e38f);
  const float t = __uint_as_float((__float_as_uint(__fmul_rn(a, 1.0f / 6.0f)) + 0x4000u) & 0xFFFF8000u);
  const float q = __fmaf_rn(__fmaf_rn(-6.0f, t, a), 1.9f / 6.0f, t);
  uint32_t r;
  asm("{\n\t.reg .b16 s;\n\tcvt.rn.satfinite.e4m3x2.f32 s, %1, %1;\n\tcvt.u32.u16 %0, s;\n\t}" : "=r"(r) : "f"(q));
  return m >= 0x7F800000u ? mx_nan_scale<FMT>() : (int)(r & 0x7F);
}

// A block's step, the value of code 1.0: scale times a power of two (the tensor scale, or a unit in
// which the block's values are held), and about one over it.
struct MxStep {
  float s, inv;
};
template <int FMT> __device__ __forceinline__ MxStep mx_step(int byte, float times) {
  MxStep st;
  st.s = __fmul_rn(mx_scale_value<FMT>(byte), times);
  if (FMT == kMXFP4) {   // a power of two (2^-127 has the field 0): its inverse is one too
    st.inv = __uint_as_float((uint32_t)(254 - (int)(__float_as_uint(st.s) >> 23)) << 23);
  } else {
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(st.inv) : "f"(st.s));
    if (!(st.s > 0.0f)) st.inv = 0.0f;   // a scale of zero: every code is zero
  }
  return st;
}

// A pair of values over a block's step, moved so that rounding to e2m1 gives what the exact quotient
// would.
//   MXFP4: v / 2^e is exact, so the conversion's rounding is the only one.
//   NVFP4: v / s is not.  t is a multiple of 1/4 next to the approximate quotient, and every border
//   between two e2m1 values is such a multiple.  t s is exact (t has at most 5 bits where a border can
//   lie, s has 4) and r = v - t s has the right sign, so t + 1.9 r / s, which stays within a quarter of
//   t, is on the side of t that v is on, and is t itself on a tie.  Quotients past 2^21, which only a
//   saturated scale leaves, lose the quarter but not that they saturate.
template <int FMT> __device__ __forceinline__ float2 mx_quotient(float2 v, const MxStep& st) {
  const float2 inv = make_float2(st.inv, st.inv);
  if (FMT == kMXFP4) return __fmul2_rn(v, inv);
  constexpr float kQuarter = 3145728.0f;   // 1.5 * 2^21: adding it rounds to a multiple of 1/4
  const float2 t = __fadd2_rn(__ffma2_rn(v, inv, make_float2(kQuarter, kQuarter)), make_float2(-kQuarter, -kQuarter));
  const float2 r = __ffma2_rn(t, make_float2(-st.s, -st.s), v);
  return __ffma2_rn(r, make_float2(1.9f * st.inv, 1.9f * st.inv), t);
}
// Codes of H pairs of values against a block's step, eight to a word.
template <int FMT, int H>
__device__ __forceinline__ void mx_codes(const float2 (&v)[H], const MxStep& st, uint32_t (&code)[H / 4]) {
  float2 q[H];
#pragma unroll
  for (int i = 0; i < H; i++) q[i] = mx_quotient<FMT>(v[i], st);
#pragma unroll
  for (int i = 0; i < H / 4; i++) code[i] = e2m1x8(q + 4 * i);
}
// A pair of quotients rounded to e2m1.
__device__ __forceinline__ float2 e2m1_round(float2 q) {
  uint32_t h;
  asm("{\n\t.reg .b8 c;\n\tcvt.rn.satfinite.e2m1x2.f32 c, %2, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}"
      : "=r"(h)
      : "f"(q.x), "f"(q.y));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

}  // namespace cpk
