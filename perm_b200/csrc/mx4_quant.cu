// Quantisation to microscaled 4-bit operands and back (layout and rounding: mx4_format.cuh), and
// the GGUF MXFP4 container.
//
// Bound by memory: a bf16 activation matrix costs 2 bytes a value to read and 17/32 or 9/16 to
// write.  A lane takes 8 columns (16 of a two-byte type to MXFP4, so that more bytes are in flight) of up to four
// rows 32 apart: those rows' scale bytes are neighbours in the scale tile, so a group of four blocks
// leaves as one 16-byte store, and the four rows' loads are in flight together.
//
// Importance-weighted scales.  For weights with column weights qw a block tries several scales
// and keeps the one with the least sum of qw (x - q s)^2: MXFP4 the exponents e, e + 1 and
// e - 1, NVFP4 the codes c, c + 1, c - 1, c + 2, c - 2, c + 3, c + 4, c + 5 (c + 4 and c + 5
// map the maximum to 4 instead of 6).  Ties go to the first.  The choice is defined by the sums in 64
// bits; float32 sums decide it unless two candidates are within 2^-16 of each other (their
// error is below 2^-19), and only then are the sums formed again in 64 bits.
#include <cuda_runtime.h>
#include <type_traits>
#include "kquant_kernels.h"
#include "mx4_format.cuh"

namespace cpk {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// Eight consecutive values of a row, in pairs; left = values of the row from here on (may be <= 0).
// Returns the largest magnitude's bits.
template <typename T>
__device__ __forceinline__ uint32_t load8(const T* p, int64_t left, bool vec, float2 (&v)[4]) {
  if (vec && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w), v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
    } else {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {   // a bf16 is the upper half of its float32
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xFFFF0000u));
        const uint32_t m = __vmaxu2(__vmaxu2(u[0] & 0x7FFF7FFFu, u[1] & 0x7FFF7FFFu),
                                    __vmaxu2(u[2] & 0x7FFF7FFFu, u[3] & 0x7FFF7FFFu));
        return max(m & 0xFFFF0000u, m << 16);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      v[i] = make_float2(2 * i < left ? to_f32(p[2 * i]) : 0.0f, 2 * i + 1 < left ? to_f32(p[2 * i + 1]) : 0.0f);
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; i++)
    m = max(m, max(__float_as_uint(v[i].x) & 0x7FFFFFFFu, __float_as_uint(v[i].y) & 0x7FFFFFFFu));
  return m;
}

template <int FMT> __host__ __device__ constexpr int mx_candidates() { return FMT == kMXFP4 ? 3 : 8; }
template <int FMT> __device__ __forceinline__ int mx_candidate(int first, int c) {
  constexpr int kMx[3] = {0, 1, -1};
  constexpr int kNv[8] = {0, 1, -1, 2, -2, 3, 4, 5};
  const int b = first + (FMT == kMXFP4 ? kMx[c < 3 ? c : 0] : kNv[c]);
  return min(max(b, 0), FMT == kMXFP4 ? 253 : 126);
}
// The step of candidate c (MXFP4: the first's, its double and its half; `first` is at least 1 there).
template <int FMT> __device__ __forceinline__ MxStep candidate_step(const MxStep& st, int first, int c, float times) {
  if (FMT == kNVFP4) return mx_step<FMT>(mx_candidate<FMT>(first, c), times);
  const float k = c == 0 ? 1.0f : c == 1 ? 2.0f : 0.5f;
  return MxStep{__fmul_rn(st.s, k), __fmul_rn(st.inv, 1.0f / k)};
}

// Sum over the lanes of a block.
template <int LANES, typename T> __device__ __forceinline__ T block_sum(T e) {
#pragma unroll
  for (int o = 1; o < LANES; o *= 2) e += __shfl_xor_sync(0xffffffffu, e, o);
  return e;
}

// H pairs by groups of four.
template <typename T, int H>
__device__ __forceinline__ uint32_t load_pairs(const T* p, int64_t left, bool vec, float2 (&v)[H]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < H; i += 4) m = max(m, load8(p + 2 * i, left - 2 * i, vec, *reinterpret_cast<float2(*)[4]>(&v[i])));
  return m;
}

// Scale byte and codes of a block (H pairs per lane, `top` the largest of them as bits).
template <int FMT, bool IMAT, int H>
__device__ __forceinline__ void quantize_block(float2 (&v)[H], uint32_t top, const float2 (&w)[H], float tensor_scale,
                                               float inv_tensor_scale, int& byte, uint32_t (&code)[H / 4]) {
  constexpr int LANES = mx_block<FMT>() / (2 * H);
  const uint32_t m = mx_block_max<LANES>(top);
  byte = mx_first_scale<FMT>(m, inv_tensor_scale);
  const bool finite = m < 0x7F800000u;   // else the scale byte is NaN and the block decodes to NaN
  if constexpr (!IMAT) {
    mx_codes<FMT, H>(v, mx_step<FMT>(byte, tensor_scale), code);
  } else {
    constexpr int C = mx_candidates<FMT>();
    const int first = byte;
    // values and steps in units of the block's maximum (a power of two), so that squares neither vanish
    // nor overflow.  Not searched, and not in such units, are a block with scale byte 0 (all but empty: NVFP4's
    // step in units of so small a maximum may be infinite) and one of NVFP4 that is past 2^100 tensor
    // scales (saturated throughout; its step may vanish).
    float unit = __uint_as_float((uint32_t)min(max(254 - (int)(m >> 23), 1), 253) << 23);
    const bool search = finite && first > 0 && (FMT == kMXFP4 || __fmul_rn(tensor_scale, unit) >= 0x1p-100f);
    unit = search ? unit : 1.0f;
    const float times = __fmul_rn(tensor_scale, unit);
    float err[C];
    const MxStep step0 = mx_step<FMT>(first, times);
#pragma unroll
    for (int i = 0; i < H; i++) v[i] = __fmul2_rn(v[i], make_float2(unit, unit));
#pragma unroll
    for (int c = 0; c < C; c++) {
      const MxStep st = candidate_step<FMT>(step0, first, c, times);
      const float2 ms = make_float2(-st.s, -st.s);
      float2 e = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < H; i++) {
        const float2 d = __ffma2_rn(e2m1_round(mx_quotient<FMT>(v[i], st)), ms, v[i]);
        e = __ffma2_rn(__fmul2_rn(w[i], d), d, e);
      }
      err[c] = block_sum<LANES>(e.x + e.y);
    }
    int pick = 0;
    float best = err[0];
#pragma unroll
    for (int c = 1; c < C; c++)
      if (err[c] < best) best = err[c], pick = c;
    // near: some other candidate is as good as the float32 sums can tell, or the sums are out of
    // float32's range
    bool near = !(best > 1e-30f && best < 1e30f);
#pragma unroll
    for (int c = 0; c < C; c++) near |= c != pick && err[c] <= best * 1.0000153f;
    near = near && search;
    if (__any_sync(0xffffffffu, near)) {
      double bd = 0.0;
      int pd = 0;
#pragma unroll 1
      for (int c = 0; c < C; c++) {
        const MxStep st = candidate_step<FMT>(step0, first, c, times);
        double e = 0.0;
#pragma unroll
        for (int i = 0; i < H; i++) {
          const float2 q = e2m1_round(mx_quotient<FMT>(v[i], st));
          const double d0 = (double)v[i].x - (double)q.x * (double)st.s, d1 = (double)v[i].y - (double)q.y * (double)st.s;
          e += (double)w[i].x * (d0 * d0);
          e += (double)w[i].y * (d1 * d1);
        }
        e = block_sum<LANES>(e);
        if (c == 0 || e < bd) bd = e, pd = c;
      }
      if (near) pick = pd;
    }
    if (!search) pick = 0;
    if (pick > 0) byte = mx_candidate<FMT>(first, pick);
    mx_codes<FMT, H>(v, mx_step<FMT>(byte, times), code);
  }
#pragma unroll
  for (int i = 0; i < H / 4; i++) code[i] = finite ? code[i] : 0;
}

constexpr int kWarps = 8;

// Units (row lane r of a row tile, chunk of 64 H columns), one per warp; pitch = columns of the padded row.
template <typename T, int FMT, bool IMAT, int H>
__global__ void __launch_bounds__(32 * kWarps)
    quantize_kernel(const T* __restrict__ x, int64_t rows, int64_t n, int64_t ld, const float* __restrict__ qw,
                    float scale, float inv_scale, int chunks, int64_t pitch, int64_t units, bool vec,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int64_t unit = blockIdx.x * (int64_t)kWarps + threadIdx.x / 32;
  if (unit >= units) return;
  const int lane = threadIdx.x % 32;
  const int64_t rl = unit / chunks;                 // 32 row lanes per tile of 128 rows
  const int64_t row0 = (rl >> 5) * 128 + (rl & 31);
  const int64_t col = (unit - rl * chunks) * (64 * H) + lane * 2 * H, left = n - col;
  float2 v[4][H], w[H];
  uint32_t top[4];
#pragma unroll
  for (int j = 0; j < 4; j++) top[j] = load_pairs<T, H>(x + (row0 + 32 * j) * ld + col, row0 + 32 * j < rows ? left : 0, vec, v[j]);
  if constexpr (IMAT) load_pairs<float, H>(qw + col, left, (reinterpret_cast<uintptr_t>(qw) & 15) == 0, w);
  constexpr int LB = mx_block<FMT>() / (2 * H);   // lanes per block
  uint32_t sb[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    int byte;
    uint32_t code[H / 4];
    quantize_block<FMT, IMAT, H>(v[j], top[j], w, scale, inv_scale, byte, code);
    if (row0 + 32 * j < rows && col < pitch) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(codes + (row0 + 32 * j) * (pitch / 2) + col / 2);
      if constexpr (H == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(code[0], code[1]);
      else *dst = code[0];
    }
    // the four bytes of a group of four blocks, gathered into its first lane
    uint32_t b = (uint32_t)byte;
    b |= __shfl_down_sync(0xffffffffu, b, LB) << 8;
    b |= __shfl_down_sync(0xffffffffu, b, 2 * LB) << 16;
    sb[j] = b;
  }
  if (lane % (4 * LB) == 0 && col < pitch) {
    const int64_t groups = pitch / (4 * mx_block<FMT>()), g = col / (4 * mx_block<FMT>());
    *reinterpret_cast<uint4*>(scales + ((row0 >> 7) * groups + g) * 512 + (row0 & 31) * 16) =
        make_uint4(sb[0], sb[1], sb[2], sb[3]);
  }
}

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }

// A lane takes 16 bytes of results at a time (8 or 4 values), so that a warp's stores are whole lines: two
// neighbouring stores of 16 bytes per lane took 64 us for 14336 x 4096 float32.
template <typename T, int FMT>
__global__ void __launch_bounds__(32 * kWarps)
    dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows, int64_t n,
                      float scale, int chunks, int64_t units, bool vec, T* __restrict__ out, int64_t ld) {
  const int64_t unit = blockIdx.x * (int64_t)kWarps + threadIdx.x / 32;
  if (unit >= units) return;
  constexpr int G = 16 / sizeof(T), B = mx_block<FMT>();
  const int64_t rl = unit / chunks;
  const int chunk = (int)(unit - rl * chunks);
  const int64_t row0 = (rl >> 5) * 128 + (rl & 31);
  const int64_t pitch = (int64_t)chunks * 128, groups = (int64_t)chunks * (64 / B);
#pragma unroll
  for (int k = 0; k < 8 / G; k++) {
    const int at = k * (32 * G) + (threadIdx.x % 32) * G;   // in the chunk of 256 columns
    const int64_t col = (int64_t)chunk * 256 + at, left = n - col;
    if (left <= 0) return;
    const uint4 sw = __ldg(reinterpret_cast<const uint4*>(
        scales + ((row0 >> 7) * groups + (int64_t)chunk * (64 / B) + at / (4 * B)) * 512 + (row0 & 31) * 16));
    const uint32_t sj[4] = {sw.x, sw.y, sw.z, sw.w};
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint8_t* src = codes + (row0 + 32 * j) * pitch + col / 2;
      c[j] = row0 + 32 * j >= rows ? 0
             : G == 8              ? __ldg(reinterpret_cast<const uint32_t*>(src))
                                   : __ldg(reinterpret_cast<const uint16_t*>(src));
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t row = row0 + 32 * j;
      if (row >= rows) break;
      const float s = mx_scale_value<FMT>((sj[j] >> (8 * (at / B % 4))) & 0xFF);
      T o[G];
#pragma unroll
      for (int i = 0; i < G / 2; i++) {
        const float2 q = e2m1x2_value(c[j] >> (8 * i));
        // q s is exact, so the tensor scale's product is the only rounding before the type's own
        put(o + 2 * i, __fmul_rn(__fmul_rn(q.x, s), scale));
        put(o + 2 * i + 1, __fmul_rn(__fmul_rn(q.y, s), scale));
      }
      T* p = out + row * ld + col;
      if (vec && left >= G) {
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(o);
      } else {
#pragma unroll
        for (int i = 0; i < G; i++)
          if (i < left) p[i] = o[i];
      }
    }
  }
}

// ---------------------------------------------------------------------------- GGUF container
// Blocks of 32: the scale byte, then 16 bytes whose low halves are values 0-15 and whose high
// halves are values 16-31.  Blocks follow one another through the whole tensor, so the kernels
// take them flat, 256 per CTA: 4352 bytes, staged in shared memory and moved 16 bytes at a time.
constexpr int kBlkBytes = 17, kCtaBlocks = 256;

// Nibbles of a and b interleaved into bytes a_i | b_i << 4, for i = 0..3 (lo) and 4..7 (hi).
__device__ __forceinline__ uint32_t spread16(uint32_t h) {   // 4 nibbles -> 4 bytes
  h = (h | (h << 8)) & 0x00FF00FFu;
  return (h | (h << 4)) & 0x0F0F0F0Fu;
}

template <bool IMAT>
__global__ void __launch_bounds__(256) encode_kernel(const float* __restrict__ x, int64_t nblk, int nb_row,
                                                     const float* __restrict__ qw, uint8_t* __restrict__ out) {
  __shared__ __align__(16) uint8_t stage[kCtaBlocks * kBlkBytes];
  const int64_t b0 = (int64_t)blockIdx.x * kCtaBlocks;
  const int t = threadIdx.x, l4 = t & 3;
  const uint32_t in_row = IMAT ? (uint32_t)(b0 % nb_row) : 0;   // the first block's place in its row
  float2 v[4][4];
  uint32_t top[4];
#pragma unroll
  for (int p = 0; p < 4; p++) {
    const int64_t b = b0 + p * 64 + (t >> 2);
    top[p] = load8(x + b * 32 + l4 * 8, b < nblk ? 8 : 0, true, v[p]);
  }
#pragma unroll
  for (int p = 0; p < 4; p++) {
    const int lb = p * 64 + (t >> 2);
    const int64_t b = b0 + lb;
    float2 w[4];
    if constexpr (IMAT) load8(qw + (int64_t)((in_row + lb) % (uint32_t)nb_row) * 32 + l4 * 8, b < nblk ? 8 : 0, true, w);
    int byte;
    uint32_t code[1];
    quantize_block<kMXFP4, IMAT, 4>(v[p], top[p], w, 1.0f, 1.0f, byte, code);
    const uint32_t c = code[0];
    const uint32_t other = __shfl_xor_sync(0xffffffffu, c, 2);   // values 16 further (lanes 0, 1)
    if (l4 < 2) {
      const uint32_t lo = spread16(c & 0xFFFF) | spread16(other & 0xFFFF) << 4;
      const uint32_t hi = spread16(c >> 16) | spread16(other >> 16) << 4;
      uint8_t* q = stage + lb * kBlkBytes + 1 + l4 * 8;
#pragma unroll
      for (int i = 0; i < 4; i++) q[i] = (uint8_t)(lo >> (8 * i)), q[4 + i] = (uint8_t)(hi >> (8 * i));
      if (l4 == 0) stage[lb * kBlkBytes] = (uint8_t)byte;
    }
  }
  __syncthreads();
  const int64_t left = nblk - b0;
  const int bytes = (int)(left < kCtaBlocks ? left : kCtaBlocks) * kBlkBytes;
  uint8_t* dst = out + b0 * kBlkBytes;
  for (int i = t; i < bytes / 16; i += 256) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(stage)[i];
  if (t < bytes % 16) dst[bytes / 16 * 16 + t] = stage[bytes / 16 * 16 + t];
}

// Brings a CTA's blocks into shared memory.
__device__ __forceinline__ int load_blocks(const uint8_t* __restrict__ raw, int64_t nblk, int64_t b0, uint8_t* stage) {
  const int64_t left = nblk - b0;
  const int bytes = (int)(left < kCtaBlocks ? left : kCtaBlocks) * kBlkBytes;
  const uint8_t* src = raw + b0 * kBlkBytes;
  for (int i = threadIdx.x; i < bytes / 16; i += 256)
    reinterpret_cast<uint4*>(stage)[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
  if ((int)threadIdx.x < bytes % 16) stage[bytes / 16 * 16 + threadIdx.x] = src[bytes / 16 * 16 + threadIdx.x];
  __syncthreads();
  return bytes / kBlkBytes;
}

// Values 4 l .. 4 l + 3 of staged block lb.  Its four bytes start anywhere, so they come out of two
// aligned words.
__device__ __forceinline__ float4 block_values(const uint8_t* stage, int lb, int l) {
  const uint32_t at = lb * kBlkBytes + 1 + (l & 3) * 4;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(stage) + at / 4;
  const uint32_t c = (__funnelshift_r(w[0], w[1], 8 * (at & 3)) >> (l >= 4 ? 4 : 0)) & 0x0F0F0F0Fu;
  const uint32_t two = c | (c >> 4);   // bytes 0 and 2: codes 0, 1 and 2, 3
  const float s = e8m0_value(stage[lb * kBlkBytes]);
  const float2 a = e2m1x2_value(two), b = e2m1x2_value(two >> 16);
  return make_float4(__fmul_rn(a.x, s), __fmul_rn(a.y, s), __fmul_rn(b.x, s), __fmul_rn(b.y, s));
}

__global__ void __launch_bounds__(256) decode_kernel(const uint8_t* __restrict__ raw, int64_t nblk,
                                                     float* __restrict__ out) {
  __shared__ __align__(16) uint8_t stage[kCtaBlocks * kBlkBytes + 16];
  const int64_t b0 = (int64_t)blockIdx.x * kCtaBlocks;
  const int n = load_blocks(raw, nblk, b0, stage);
  const int t = threadIdx.x;
#pragma unroll
  for (int p = 0; p < 8; p++) {
    const int lb = p * 32 + (t >> 3);
    if (lb < n) reinterpret_cast<float4*>(out + b0 * 32)[p * 256 + t] = block_values(stage, lb, t & 7);
  }
}

// *err += sum of w (x - value)^2 in 64 bits, one atomic per CTA.
__global__ void __launch_bounds__(256) weighted_err_kernel(const uint8_t* __restrict__ raw, const float* __restrict__ x,
                                                           const float* __restrict__ w, int64_t nblk, int nb_row,
                                                           double* __restrict__ err) {
  __shared__ __align__(16) uint8_t stage[kCtaBlocks * kBlkBytes + 16];
  __shared__ double part[8];
  const int64_t b0 = (int64_t)blockIdx.x * kCtaBlocks;
  const int n = load_blocks(raw, nblk, b0, stage);
  const uint32_t in_row = (uint32_t)(b0 % nb_row);
  const int t = threadIdx.x;
  double e = 0.0;
  for (int p = 0; p < 8; p++) {
    const int lb = p * 32 + (t >> 3);
    if (lb >= n) break;
    const float4 v = block_values(stage, lb, t & 7);
    const float4 y = __ldg(reinterpret_cast<const float4*>(x + b0 * 32) + p * 256 + t);
    const float4 g = w ? __ldg(reinterpret_cast<const float4*>(w + (int64_t)((in_row + lb) % (uint32_t)nb_row) * 32) + (t & 7))
                       : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    const double d[4] = {(double)v.x - y.x, (double)v.y - y.y, (double)v.z - y.z, (double)v.w - y.w};
    e += d[0] * d[0] * g.x + d[1] * d[1] * g.y + d[2] * d[2] * g.z + d[3] * d[3] * g.w;
  }
  for (int o = 16; o; o >>= 1) e += __shfl_down_sync(0xffffffffu, e, o);
  if (t % 32 == 0) part[t / 32] = e;
  __syncthreads();
  if (t == 0) {
    for (int i = 1; i < 8; i++) e += part[i];
    atomicAdd(err, e);
  }
}

__host__ __device__ inline int64_t tile_rows(int64_t rows) { return (rows + 127) / 128 * 128; }

// Container -> operand: one thread per block of the padded row (blocks past n, and the scale bytes of the rows
// that fill the last tile: zero).
__global__ void __launch_bounds__(256) unpack_kernel(const uint8_t* __restrict__ raw, int64_t nrow, int nb_row, int nb_pad,
                                                     uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
  const int64_t row = i / nb_pad;
  if (row >= tile_rows(nrow)) return;
  const int b = (int)(i - row * nb_pad);
  if (row >= nrow) {
    scales[mx_scale_offset(row, b, nb_pad / 4)] = 0;
    return;
  }
  uint32_t o[4] = {0, 0, 0, 0};
  uint8_t s = 0;
  if (b < nb_row) {
    const uint8_t* src = raw + (row * nb_row + b) * kBlkBytes;
    s = src[0];
#pragma unroll
    for (int j = 0; j < 16; j++) {   // value j: low half, nibble j of the row; value j + 16: high half
      const uint32_t q = src[1 + j];
      o[j >> 3] |= (q & 15) << (4 * (j & 7));
      o[2 + (j >> 3)] |= (q >> 4) << (4 * (j & 7));
    }
  }
  *reinterpret_cast<uint4*>(codes + i * 16) = make_uint4(o[0], o[1], o[2], o[3]);
  scales[mx_scale_offset(row, b, nb_pad / 4)] = s;
}

// Row lanes that hold a row.
int64_t row_lanes(int64_t rows) { return rows / 128 * 32 + (rows % 128 < 32 ? rows % 128 : 32); }

template <typename T, int FMT, bool IMAT>
int quantize_typed(const T* x, int64_t rows, int64_t n, int64_t ld, const float* qw, float scale, uint8_t* codes,
                   uint8_t* scales, cudaStream_t stream) {
  // 8192 x 4096 bf16 to MXFP4: 16.5 us with H = 8, 20.8 with 4; to NVFP4, whose rounding keeps more values in
  // registers, 22 us with either.
  constexpr int H = sizeof(T) == 2 && FMT == kMXFP4 && !IMAT ? 8 : 4;
  const int64_t pitch = (n + 255) / 256 * 256;
  const int chunks = (int)((pitch + 64 * H - 1) / (64 * H));
  const int64_t units = tile_rows(rows) / 4 * chunks;   // all row lanes of a tile: their scale bytes are zero past the last row
  const unsigned grid = (unsigned)((units + kWarps - 1) / kWarps);
  const bool vec = ((uintptr_t)x & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
  quantize_kernel<T, FMT, IMAT, H><<<grid, 32 * kWarps, 0, stream>>>(x, rows, n, ld, qw, scale, 1.0f / scale, chunks, pitch,
                                                                    units, vec, codes, scales);
  note_launch();
  return 0;
}

template <typename T>
int quantize_format(int fmt, const T* x, int64_t rows, int64_t n, int64_t ld, const float* qw, float scale, uint8_t* codes,
                    uint8_t* scales, cudaStream_t stream) {
  if (fmt == kMXFP4)
    return qw ? quantize_typed<T, kMXFP4, true>(x, rows, n, ld, qw, scale, codes, scales, stream)
              : quantize_typed<T, kMXFP4, false>(x, rows, n, ld, qw, scale, codes, scales, stream);
  return qw ? quantize_typed<T, kNVFP4, true>(x, rows, n, ld, qw, scale, codes, scales, stream)
            : quantize_typed<T, kNVFP4, false>(x, rows, n, ld, qw, scale, codes, scales, stream);
}

template <typename T> int dequantize_typed(const Mx4View& v, float scale, T* out, int64_t ld, cudaStream_t stream) {
  const int chunks = (int)((v.n + 255) / 256);
  const int64_t units = row_lanes(v.rows) * chunks;
  const unsigned grid = (unsigned)((units + kWarps - 1) / kWarps);
  const bool vec = ((uintptr_t)out & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
  if (v.fmt == kMXFP4)
    dequantize_kernel<T, kMXFP4><<<grid, 32 * kWarps, 0, stream>>>(v.codes, v.scales, v.rows, v.n, scale, chunks, units, vec, out, ld);
  else
    dequantize_kernel<T, kNVFP4><<<grid, 32 * kWarps, 0, stream>>>(v.codes, v.scales, v.rows, v.n, scale, chunks, units, vec, out, ld);
  note_launch();
  return 0;
}

}  // namespace

int launch_mx4_quantize(int fmt, int dtype, const void* x, int64_t rows, int64_t n, int64_t ld, const float* qw,
                        float scale, uint8_t* codes, uint8_t* scales, cudaStream_t stream) {
  if (rows == 0) return 0;
  if (dtype == kMxBF16)
    return quantize_format(fmt, static_cast<const __nv_bfloat16*>(x), rows, n, ld, qw, scale, codes, scales, stream);
  if (dtype == kMxF16)
    return quantize_format(fmt, static_cast<const __half*>(x), rows, n, ld, qw, scale, codes, scales, stream);
  return quantize_format(fmt, static_cast<const float*>(x), rows, n, ld, qw, scale, codes, scales, stream);
}

int launch_mx4_dequantize(const Mx4View& v, float scale, int dtype, void* out, int64_t ld, cudaStream_t stream) {
  if (v.rows == 0) return 0;
  if (dtype == kMxBF16) return dequantize_typed(v, scale, static_cast<__nv_bfloat16*>(out), ld, stream);
  if (dtype == kMxF16) return dequantize_typed(v, scale, static_cast<__half*>(out), ld, stream);
  return dequantize_typed(v, scale, static_cast<float*>(out), ld, stream);
}

int launch_mx4_encode(const float* x, int64_t nrow, int64_t n, const float* qw, uint8_t* out, cudaStream_t stream) {
  const int64_t nblk = nrow * (n / 32);
  if (nblk == 0) return 0;
  const unsigned grid = (unsigned)((nblk + kCtaBlocks - 1) / kCtaBlocks);
  if (qw) encode_kernel<true><<<grid, 256, 0, stream>>>(x, nblk, (int)(n / 32), qw, out);
  else encode_kernel<false><<<grid, 256, 0, stream>>>(x, nblk, (int)(n / 32), qw, out);
  note_launch();
  return 0;
}

int launch_mx4_decode(const uint8_t* raw, int64_t nrow, int64_t n, float* out, cudaStream_t stream) {
  const int64_t nblk = nrow * (n / 32);
  if (nblk == 0) return 0;
  decode_kernel<<<(unsigned)((nblk + kCtaBlocks - 1) / kCtaBlocks), 256, 0, stream>>>(raw, nblk, out);
  note_launch();
  return 0;
}

int launch_mx4_weighted_err(const uint8_t* raw, const float* x, const float* w, int64_t nrow, int64_t n, double* err,
                            cudaStream_t stream) {
  const int64_t nblk = nrow * (n / 32);
  if (nblk == 0) return 0;
  weighted_err_kernel<<<(unsigned)((nblk + kCtaBlocks - 1) / kCtaBlocks), 256, 0, stream>>>(raw, x, w, nblk, (int)(n / 32), err);
  note_launch();
  return 0;
}

int launch_mx4_unpack(const uint8_t* raw, int64_t nrow, int64_t n, uint8_t* codes, uint8_t* scales,
                      cudaStream_t stream) {
  if (nrow == 0) return 0;
  const int nb = (int)(n / 32), nbp = (int)((n + 255) / 256 * 8);
  const int64_t total = tile_rows(nrow) * nbp;
  unpack_kernel<<<(unsigned)((total + 255) / 256), 256, 0, stream>>>(raw, nrow, nb, nbp, codes, scales);
  note_launch();
  return 0;
}

}  // namespace cpk
