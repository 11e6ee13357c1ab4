// Internal launcher declarations for the microscaled 4-bit operators.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace cpk {

enum Mx4Format : int { kMXFP4 = 39, kNVFP4 = 40 };        // GGML type ids
enum Mx4Dtype : int { kMxBF16 = 0, kMxF16 = 1, kMxF32 = 2 };

// A 4-bit operand in device memory (layout in mx4_format.cuh).
struct Mx4View {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t rows, n;
  int fmt;
};

inline int64_t mx4_pitch(int64_t n) { return (n + 255) / 256 * 128; }   // code bytes per row
inline int64_t mx4_scale_bytes(int fmt, int64_t rows, int64_t n) {
  return (rows + 127) / 128 * 128 * ((n + 255) / 256 * (fmt == kMXFP4 ? 8 : 16));
}

int launch_mx4_quantize(int fmt, int dtype, const void* x, int64_t rows, int64_t n, int64_t ld, const float* qw,
                        float scale, uint8_t* codes, uint8_t* scales, cudaStream_t stream);
// out: rows ld elements apart.
int launch_mx4_dequantize(const Mx4View& v, float scale, int dtype, void* out, int64_t ld, cudaStream_t stream);
// GGUF MXFP4 container (17-byte blocks of 32): encode, decode, weighted error, and to the operand.
int launch_mx4_encode(const float* x, int64_t nrow, int64_t n, const float* qw, uint8_t* out, cudaStream_t stream);
int launch_mx4_decode(const uint8_t* raw, int64_t nrow, int64_t n, float* out, cudaStream_t stream);
int launch_mx4_weighted_err(const uint8_t* raw, const float* x, const float* w, int64_t nrow, int64_t n, double* err,
                            cudaStream_t stream);
int launch_mx4_unpack(const uint8_t* raw, int64_t nrow, int64_t n, uint8_t* codes, uint8_t* scales,
                      cudaStream_t stream);

// y[t][r] = alpha * sum_k a[t][k] w[r][k]
int launch_mx4_matmul(const Mx4View& a, const Mx4View& w, float alpha, int dtype, void* y, cudaStream_t stream);

// transpose == 0: y[t][r] = alpha * sum_k x[t][k] w[r][k]   (x [T, w.n],    y [T, w.rows])
// transpose == 1: y[t][k] = alpha * sum_r x[t][r] w[r][k]   (x [T, w.rows], y [T, w.n])
// aligned: x's rows start on 16-byte boundaries.
size_t mx4_linear_workspace_bytes(int dtype, int64_t T, int64_t rows, int64_t n, int aligned, int transpose);
int launch_mx4_linear(int dtype, const void* x, int64_t T, int64_t ld, int aligned, const Mx4View& w, float alpha,
                      int transpose, void* y, void* ws, cudaStream_t stream);

// The first form for a few tokens (mx4_stream.cu), and whether it takes these sizes.
bool mx4_stream_applies(int dtype, int64_t T, int64_t rows, int64_t n);
size_t mx4_stream_workspace_bytes(int dtype, int64_t T, int64_t rows, int64_t n);
int launch_mx4_stream(int dtype, const void* x, int64_t T, int64_t ld, int aligned, const Mx4View& w, float alpha, void* y,
                      void* ws, cudaStream_t stream);

// Bound of every wait of the calling thread's next product, and (failure-path tests) the load step that each CTA
// leaves out of it; -1: none.
struct Mx4Waits {
  unsigned long long ns;
  int skip;
};
Mx4Waits mx4_take_waits();

// Status words of the products' bounded waits (read and cleared; synchronises the stream).
int mx4_matmul_status(cudaStream_t stream, int* status);
int mx4_linear_status(cudaStream_t stream, int* status);
int mx4_stream_status(cudaStream_t stream, int* status);

}  // namespace cpk
