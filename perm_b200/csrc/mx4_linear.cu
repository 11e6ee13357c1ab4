// Products with 4-bit operands: a 64 x 64 output tile per CTA, operands decoded to float32 in shared
// memory 32 deep, 4 x 4 outputs per thread.
#include <cuda_runtime.h>
#include "kquant_kernels.h"
#include "mx4_format.cuh"

namespace cpk {
namespace {

struct Packed {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t rows, n;
};
template <int FMT> __device__ __forceinline__ float packed_at(const Packed& p, int64_t r, int64_t k) {
  if (r >= p.rows || k >= p.n) return 0.0f;
  const int64_t chunks = (p.n + 255) / 256;
  const uint32_t b = p.codes[r * chunks * 128 + (k >> 1)];
  const float q = e2m1x2_value((b >> (4 * (k & 1))) & 15).x;
  constexpr int B = mx_block<FMT>();
  return q * mx_scale_value<FMT>(p.scales[mx_scale_offset(r, k / B, chunks * (64 / B))]);
}
__device__ __forceinline__ float dense_at(const void* x, int dtype, int64_t i) {
  return dtype == kMxBF16  ? __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i])
         : dtype == kMxF16 ? __half2float(static_cast<const __half*>(x)[i])
                           : static_cast<const float*>(x)[i];
}
__device__ __forceinline__ void put(void* y, int dtype, int64_t i, float v) {
  if (dtype == kMxBF16) static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
  else if (dtype == kMxF16) static_cast<__half*>(y)[i] = __float2half_rn(v);
  else static_cast<float*>(y)[i] = v;
}

template <int FMT>
__global__ void __launch_bounds__(256) product_kernel(Packed a, const void* x, int dtype_x, int64_t T, int64_t ld,
                                                      Packed w, int transpose, float alpha, int dtype, void* y) {
  __shared__ float sx[32][65], sw[32][65];
  const int64_t out = transpose ? w.n : w.rows, K = transpose ? w.rows : w.n;
  const int64_t o0 = (int64_t)blockIdx.x * 64, t0 = (int64_t)blockIdx.y * 64;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += 32) {
    for (int i = threadIdx.x; i < 2048; i += 256) {
      const int k = i % 32, j = i / 32;
      const int64_t t = t0 + j, o = o0 + j, kk = k0 + k;
      sx[k][j] = t >= T || kk >= K ? 0.0f : x ? dense_at(x, dtype_x, t * ld + kk) : packed_at<FMT>(a, t, kk);
      sw[k][j] = transpose ? packed_at<FMT>(w, kk, o) : packed_at<FMT>(w, o, kk);
    }
    __syncthreads();
    for (int k = 0; k < 32; k++)
      for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) acc[i][j] += sx[k][ty + 16 * i] * sw[k][tx + 16 * j];
    __syncthreads();
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) {
      const int64_t t = t0 + ty + 16 * i, o = o0 + tx + 16 * j;
      if (t < T && o < out) put(y, dtype, t * out + o, alpha * acc[i][j]);
    }
}

int launch_product(const Packed& a, const void* x, int dtype_x, int64_t T, int64_t ld, const Mx4View& w, int transpose,
                   float alpha, int dtype, void* y, cudaStream_t stream) {
  const int64_t out = transpose ? w.n : w.rows;
  const dim3 grid((unsigned)((out + 63) / 64), (unsigned)((T + 63) / 64));
  const Packed pw{w.codes, w.scales, w.rows, w.n};
  if (w.fmt == kMXFP4) product_kernel<kMXFP4><<<grid, 256, 0, stream>>>(a, x, dtype_x, T, ld, pw, transpose, alpha, dtype, y);
  else product_kernel<kNVFP4><<<grid, 256, 0, stream>>>(a, x, dtype_x, T, ld, pw, transpose, alpha, dtype, y);
  note_launch();
  return 0;
}

}  // namespace

size_t mx4_linear_workspace_bytes(int, int64_t, int64_t, int64_t, int64_t, int, int) { return 0; }

int launch_mx4_linear(int dtype, const void* x, int64_t T, int64_t ld, const Mx4View& w, float alpha, int transpose,
                      void* y, void*, cudaStream_t stream) {
  return launch_product({}, x, dtype, T, ld, w, transpose, alpha, dtype, y, stream);
}

}  // namespace cpk
