// y = alpha * x W^T (or x W, TR) for many tokens: W's 4-bit values decoded once to bf16 in the
// workspace (exact), then a bf16 tensor-core product on SM pairs.
//
// Decoding inside the product (mx4_linear.cu) repeats for every token tile and its stores share the shared
// memory's bandwidth with the MMAs' reads; past a few token tiles one pass that writes and reads 2
// bytes a weight is cheaper.
//
// Clusters of two CTAs take 256 (output rows) x 256 (tokens) tiles with tcgen05.mma.cta_group::2
// kind::f16.  Each CTA loads, by TMA, its 128 rows of W and, for each part of x, half of the tokens,
// 64 deep per stage; both CTAs' loads complete on the even CTA's barrier.  Two accumulators
// alternate: eight epilogue warps read a finished one into registers while the MMAs go on in the other.
// float32 results take a new accumulator every step (12 MMAs, the smallest part of x first) and sum the
// chunks in those registers, because the tensor core's own accumulation truncates: sums of positive products
// come out low by 2^-24 on average; with three steps to a chain and the largest part first it was 2^-19
// (4096 x 4096 -> 4096 348 us, was 340).
#pragma once
#include "mx4_product.cuh"

namespace cpk {
namespace dense {

constexpr int kThreads = 320;   // warps: 0 loads, 1 MMA, 2-9 epilogue (two per lane quarter, 128 columns each)
constexpr int kBox = 128 * 128;                 // 128 rows x 64, or 64 rows x 128 as two boxes: bf16
constexpr int kRing = 7 * 2 * kBox;
constexpr int kMaxStages = 7;
constexpr size_t kSmem = 1024 + kRing + 256;

struct Params {
  void* y;
  int* status;
  int64_t T, out;
  float alpha;
  int dtype;
  int parts, nst;
  int steps, chunk;     // 64-deep steps; steps of one accumulation chain
  int mtiles, tiles;
  Mx4Waits waits;
};

template <bool TR>
__global__ void __launch_bounds__(kThreads, 1)
    dense_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params prm) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + kRing);   // full, empty, acc_full[2], acc_empty[2], done
  volatile int* misc = reinterpret_cast<volatile int*>(bars + 2 * kMaxStages + 5);   // [0] tmem, [1] abort
  const int nst = prm.nst, stage_bytes = (1 + prm.parts) * kBox;
  const uint32_t ring = smem_u32(base), full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages;
  const uint32_t accf = empty0 + 8 * kMaxStages, acce = accf + 16, done = acce + 16;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = (int)cluster_rank();
  const bool leader = rank == 0;
  const int first = (int)blockIdx.x / 2, stride = (int)gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; s++) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(accf + 8 * b, 1);
      mbar_init(acce + 8 * b, 16);
    }
    mbar_init(done, 1);
    misc[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
  }
  if (warp == 1) tmem_alloc<true>(smem_u32((const void*)&misc[0]), 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // both CTAs' barriers are initialised and their tensor memory allocated
  tc_fence_after();
  const uint32_t tmem = (uint32_t)misc[0];
  volatile int* abort = &misc[1];
  const uint32_t peer_abort = peer_addr(smem_u32((const void*)&misc[1]), rank ^ 1);

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t lead_full = peer_addr(full0, 0);
      Ring rg{0, 0};
      int loads = 0;
      bool ok = true;
      for (int tile = first; ok && tile < prm.tiles; tile += stride) {
        const int m0 = tile % prm.mtiles * 256 + rank * 128, t0 = tile / prm.mtiles * 256 + rank * 128;
        for (int s = 0; s < prm.steps; s++, loads++) {
          if (loads >= nst && !mbar_wait(empty0 + 8 * rg.st, rg.ph ^ 1, abort, prm.waits.ns)) {
            ok = false;
            break;
          }
          if (loads != prm.waits.skip) {
            const uint32_t fb = lead_full + 8 * rg.st, sw = ring + rg.st * stage_bytes;
            if (leader) mbar_expect_tx(full0 + 8 * rg.st, 2 * stage_bytes);
            if (TR) {
              tma_load_pair(sw, &map_w, m0, s * 64, fb);
              tma_load_pair(sw + kBox / 2, &map_w, m0 + 64, s * 64, fb);
            } else {
              tma_load_pair(sw, &map_w, s * 64, m0, fb);
            }
            for (int p = 0; p < prm.parts; p++)
              tma_load_pair(sw + (1 + p) * kBox, &map_x, s * 64, (int)(p * prm.T) + t0, fb);
          }
          rg.advance(nst);
        }
      }
      if (!ok) fail_pair(abort, peer_abort, prm.status);
      // every load issued lands before the CTA goes on: the even CTA sees its full barriers, the
      // odd one the MMAs that consumed its loads (or the wait's bound)
      for (int k = min(loads, nst); k > 0; k--) {
        rg.back(nst);
        int zero = 0;
        mbar_wait((leader ? full0 : empty0) + 8 * rg.st, rg.ph, &zero, prm.waits.ns);
      }
    }
  } else if (warp == 1) {
    if (leader) {
      // f32 accumulator, A and B bf16, A MN-major in the transposed form, N = 256, M = 256
      constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((TR ? 1u : 0u) << 15) | (32u << 17) | (16u << 24);
      const bool elected = elect_one();
      Ring rg{0, 0};
      int cg = 0;
      bool ok = true;
      for (int tile = first; ok && tile < prm.tiles; tile += stride)
        for (int g0 = 0; ok && g0 < prm.steps; cg++) {
          const int b = cg & 1, g1 = min(prm.steps, g0 + prm.chunk);
          if (cg >= 2 && !mbar_wait_warp(acce + 8 * b, ((cg >> 1) - 1) & 1, abort, prm.waits.ns)) {
            ok = false;
            break;
          }
          for (int s = g0; s < g1; s++) {
            if (!mbar_wait_warp(full0 + 8 * rg.st, rg.ph, abort, prm.waits.ns)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sw = ring + rg.st * stage_bytes;
            const uint64_t ad = TR ? sw128_desc(sw, kBox / 2, 1024) : sw128_desc(sw, 16, 1024);
            const uint64_t bd = sw128_desc(sw + kBox, 16, 1024);
            if (elected) {
              for (int p = prm.parts - 1; p >= 0; p--)   // the smallest part first: what truncation takes goes by the sum
#pragma unroll
                for (int kk = 0; kk < 4; kk++)   // 16 deep: 32 bytes of a K-major row, or 16 rows of 128
                  umma_bf16<true>(tmem + b * 256, ad + (TR ? 128 : 2) * kk, bd + p * (kBox / 16) + 2 * kk, kIdesc,
                                  (uint32_t)(s - g0) | (p ^ (prm.parts - 1)) | kk);
              umma_commit_group<true>(empty0 + 8 * rg.st);
            }
            __syncwarp();
            rg.advance(nst);
          }
          if (ok && elected) umma_commit_group<true>(accf + 8 * b);
          __syncwarp();
          g0 = g1;
        }
      if (!ok) fail_pair(abort, peer_abort, prm.status);
      if (elected) umma_commit_group<true>(done);   // all MMAs complete before tensor memory is freed
      int zero = 0;
      mbar_wait(done, 0, &zero, prm.waits.ns);
    }
  } else {
    const int q = warp & 3, hh = (warp - 2) >> 2;
    const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16) + hh * 128;
    const uint32_t lead_acce = peer_addr(acce, 0);
    int cg = 0;
    bool ok = true;
    for (int tile = first; ok && tile < prm.tiles; tile += stride) {
      float m[128];
      for (int g0 = 0; g0 < prm.steps; g0 += prm.chunk, cg++) {
        const int b = cg & 1;
        if (!mbar_wait_warp(accf + 8 * b, (cg >> 1) & 1, abort, prm.waits.ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (g0 == 0) {
          tmem_ld_cols(trow + b * 256, m);
        } else {
#pragma unroll
          for (int c = 0; c < 128; c += 16) {
            float v[16];
            tmem_ld_cols(trow + b * 256 + c, v);
#pragma unroll
            for (int e = 0; e < 16; e++) m[c + e] += v[e];
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (leader) mbar_arrive(acce + 8 * b);
          else mbar_arrive_remote(lead_acce + 8 * b);
        }
      }
      if (ok)
        store_tile<128>(m, prm.alpha, prm.y, prm.dtype, (int64_t)(tile % prm.mtiles) * 256 + rank * 128 + 32 * q, prm.out,
                        (int64_t)(tile / prm.mtiles) * 256 + hh * 128, prm.T);
    }
    if (!ok) fail_pair(abort, peer_abort, prm.status);
  }
  __syncwarp();
  __syncthreads();
  cluster_sync();   // neither CTA touches the other's memory from here on
  if (warp == 1) {
    tc_fence_after();
    tmem_free<true>(tmem, 512);
  }
}

}  // namespace dense
}  // namespace cpk
