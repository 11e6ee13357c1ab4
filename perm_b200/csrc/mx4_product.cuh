// What the tensor-core products with 4-bit operands share: results, split sums, launches.
#pragma once
#include <algorithm>
#include <atomic>
#include "ef_kernels.h"
#include "kquant_kernels.h"
#include "mx4_format.cuh"
#include "umma.cuh"

namespace cpk {

__device__ __forceinline__ void put_out(void* y, int dtype, int64_t i, float v) {
  if (dtype == kMxBF16) static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
  else if (dtype == kMxF16) static_cast<__half*>(y)[i] = __float2half_rn(v);
  else static_cast<float*>(y)[i] = v;
}

// Eight values as P bf16 parts each, in pairs: a part takes the next 8 significant bits (truncated, so no part
// overflows), so that three sum to a float32 exactly and two to an f16; of a NaN or infinity the first part
// holds it all.
template <int P> __device__ __forceinline__ void cut_bf16(float (&v)[8], uint32_t (&w)[P][4]) {
#pragma unroll
  for (int p = 0; p < P; p++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      uint32_t b = __float_as_uint(v[e]);
      const bool odd = (b & 0x7F800000u) == 0x7F800000u;
      if (odd && (b & 0x007FFFFFu)) b |= 0x00400000u;
      b >>= 16;
      v[e] = odd ? 0.0f : __fsub_rn(v[e], __uint_as_float(b << 16));
      w[p][e / 2] = e & 1 ? w[p][e / 2] | b << 16 : b;
    }
}

// Stores N accumulator columns of a warp: lane = output row (row0 + lane of rows), register = token
// (t0 + c of T); y is [T, rows].  Two-byte types: neighbouring lanes swap halves of a packed pair of
// columns, so that a lane holds two rows of one token and stores four bytes; a store instruction
// then covers two tokens x 64 bytes.  (One row and one token at a time, with the type looked up for
// each, took longer than the product.)
template <int N>
__device__ __forceinline__ void store_tile(const float (&v)[N], float alpha, void* y, int dtype, int64_t row0, int64_t rows,
                                           int64_t t0, int64_t T) {
  const int lane = threadIdx.x % 32;
  const int64_t row = row0 + lane;
  const int live = (int)min((int64_t)N, max((int64_t)0, T - t0));
  if (dtype == kMxF32) {
    float* p = static_cast<float*>(y) + t0 * rows + row;
    if (row < rows) {
#pragma unroll
      for (int c = 0; c < N; c++, p += rows)
        if (c < live) *p = alpha * v[c];
    }
    return;
  }
  const bool bf = dtype == kMxBF16;
  const int odd = lane & 1;
  const bool pairs = rows % 2 == 0 && (reinterpret_cast<uintptr_t>(y) & 3) == 0;
  const uint32_t sel = odd ? 0x3276u : 0x5410u;
  uint16_t* p = static_cast<uint16_t*>(y) + (t0 + odd) * rows + (row - odd);
#pragma unroll
  for (int c = 0; c < N; c += 2, p += 2 * rows) {
    const float a = alpha * v[c], b = alpha * v[c + 1];
    uint32_t w;
    if (bf) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    const uint32_t other = __shfl_xor_sync(0xffffffffu, w, 1);
    const uint32_t two = __byte_perm(w, other, sel);   // rows row - odd, row - odd + 1 of token c + odd
    if (pairs) {
      if (row < rows && c + odd < live) *reinterpret_cast<uint32_t*>(p) = two;
    } else if (c + odd < live) {
      if (row - odd < rows) p[0] = (uint16_t)two;
      if (row - odd + 1 < rows) p[1] = (uint16_t)(two >> 16);
    }
  }
}

// A role that gives up stops the others of its CTA and records the failure.
__device__ __forceinline__ void fail_cta(volatile int* abort, int* status) {
  *abort = 1;
  atomicOr(status, 1);
}

// A place in a ring of n stages and the parity of its current use.
struct Ring {
  int st;
  uint32_t ph;
  __device__ __forceinline__ void advance(int n) {
    if (++st == n) st = 0, ph ^= 1;
  }
  __device__ __forceinline__ void back(int n) {
    if (--st < 0) st += n, ph ^= 1;
  }
};

template <bool PAIR>
__device__ __forceinline__ void umma_bf16(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accum) {
  if (PAIR)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(ad), "l"(bd), "r"(idesc), "r"(accum)
                 : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(ad), "l"(bd), "r"(idesc), "r"(accum)
                 : "memory");
}

// Sums the partial tiles of a cluster of at most eight CTAs ([part][token][128 rows] float32 at the same place of
// every CTA's shared memory) in rank order, the smallest parts first; this CTA takes its share of the tokens, a thread four rows
// at a time: the loads across the cluster are what this costs.
template <int P = 1>
__device__ __forceinline__ void join_partials(const void* tile, int rank, int split, int cols, int64_t row0, int64_t t0,
                                              int64_t rows, float alpha, int dtype, void* y) {
  const int c0 = cols * rank / split, c1 = cols * (rank + 1) / split;
  const uint32_t at = smem_u32(tile);
  const int size = dtype == kMxF32 ? 4 : 2;
  const bool four = rows % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & (4 * size - 1)) == 0;
  for (int i = threadIdx.x + c0 * 32; i < c1 * 32; i += blockDim.x) {
    const int64_t row = row0 + (i & 31) * 4;
    if (row >= rows) continue;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int part = P - 1; part >= 0; part--) {
      float4 w[8];   // all loads ahead of the sum
#pragma unroll
      for (int p = 0; p < 8; p++)
        if (p < split) w[p] = ld_cluster_f32x4(peer_addr(at + 16 * (i + part * cols * 32), p));
#pragma unroll
      for (int p = 0; p < 8; p++)
        if (p < split) v.x += w[p].x, v.y += w[p].y, v.z += w[p].z, v.w += w[p].w;
    }
    v = make_float4(alpha * v.x, alpha * v.y, alpha * v.z, alpha * v.w);
    const int64_t to = (t0 + (i >> 5)) * rows + row;
    if (four) {
      if (dtype == kMxF32) {
        *reinterpret_cast<float4*>(static_cast<float*>(y) + to) = v;
      } else {
        uint2 o;
        if (dtype == kMxBF16) {
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o.x) : "f"(v.y), "f"(v.x));
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o.y) : "f"(v.w), "f"(v.z));
        } else {
          asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(o.x) : "f"(v.y), "f"(v.x));
          asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(o.y) : "f"(v.w), "f"(v.z));
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(y) + to) = o;
      }
    } else {
      const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (row + k < rows) put_out(y, dtype, to + k, e[k]);
    }
  }
}

// Clusters of `size` CTAs, one CTA to an SM, that fit the device at once: the SMs of a GPC do not divide evenly
// (the occupancy query gives 74, 33 and 15 on a B200).
inline int64_t cluster_slots(int size, int sms) {
  return size == 8 ? sms * 15 / 148 : size == 4 ? sms * 33 / 148 : sms / size;
}
// The split of the reduction (1, 2, 4 or 8 CTAs to a tile) with the shortest estimate, in clocks: rounds of
// `tiles` clusters, each CTA its share of `steps`, the join of a partial tile of nt tokens (measured 3600 to
// 5400 clocks for 128 tokens, 14 bytes a clock across the cluster) and the start.
inline int best_split(int64_t tiles, int steps, double step, int nt, int sms, double* clocks) {
  int best = 1;
  for (int s = 1; s <= 8 && s <= steps; s *= 2) {
    const int64_t fit = cluster_slots(s, sms) > 0 ? cluster_slots(s, sms) : 1;
    const double c = (double)((tiles + fit - 1) / fit) * ((steps + s - 1) / s * step + (s > 1 ? 1000 + 36.0 * nt : 0)) + 3500;
    if (s == 1 || c < *clocks) *clocks = c, best = s;
  }
  return best;
}

// Lets a kernel use all of an SM's shared memory (launches ask for what they need), once per device.
template <auto K> inline bool opt_in_smem() {
  static std::atomic<unsigned long long> opted{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (opted.load() & (1ull << dev)) return true;
  if (cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return false;
  opted.fetch_or(1ull << dev);
  return true;
}

// Makes the device's context current on this thread.  Tensor maps are made by the driver, which wants
// one, and a thread that has only launched through PyTorch's deferred device selection (the
// autograd engine's) may have none yet.
inline bool bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

// Tensor map of byte rows, boxes of 128 or 64 bytes swizzled over their width.
inline bool codes_map(CUtensorMap* m, const uint8_t* p, int64_t pitch, int64_t rows, int box_bytes, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)pitch, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {(cuuint32_t)box_bytes, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(p), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tensor map of scale tiles (512 bytes each, one after another), boxes of `box` tiles.
inline bool scales_map(CUtensorMap* m, const uint8_t* p, int64_t tiles, int box) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {128, (cuuint64_t)tiles};
  const cuuint64_t strides[1] = {512};
  const cuuint32_t boxes[2] = {128, (cuuint32_t)box};
  const cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<uint8_t*>(p), dims, strides, boxes, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tensor map of bf16 rows, boxes of 64 columns (128-byte swizzle).
inline bool bf16_map(CUtensorMap* m, const void* p, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Launches kernel K in clusters; 0, 4 (its shared memory was refused) or 6 (the launch was).  early: it may
// start before the launch ahead of it in the stream has finished (and waits for that itself).
template <auto K, typename... A>
inline int launch_cluster_after(bool early, int grid, int threads, size_t smem, int cluster, cudaStream_t stream, A... args) {
  if (!opt_in_smem<K>()) return 4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)cluster;
    at[n].val.clusterDim.y = 1;
    at[n++].val.clusterDim.z = 1;
  }
  if (early) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  if (cudaLaunchKernelEx(&cfg, K, args...) != cudaSuccess) return 6;
  note_launch();
  return 0;
}
template <auto K, typename... A>
inline int launch_cluster(int grid, int threads, size_t smem, int cluster, cudaStream_t stream, A... args) {
  return launch_cluster_after<K>(false, grid, threads, smem, cluster, stream, args...);
}

// Reads and clears a translation unit's status word.
template <typename S> inline int read_status_word(S& word, cudaStream_t stream, int* status) {
  int zero = 0;
  if (cudaMemcpyFromSymbolAsync(status, word, sizeof(int), 0, cudaMemcpyDeviceToHost, stream) != cudaSuccess ||
      cudaStreamSynchronize(stream) != cudaSuccess)
    return 1;
  if (*status && (cudaMemcpyToSymbolAsync(word, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream) != cudaSuccess ||
                  cudaStreamSynchronize(stream) != cudaSuccess))
    return 1;
  return 0;
}

}  // namespace cpk
