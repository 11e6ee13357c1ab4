// y = alpha * a w^T for two 4-bit operands of one format: a [T, n] (tokens), w [rows, n] (weights).
//
// Block-scaled tensor-core kernel: tcgen05.mma kind::mxf4 (e8m0 scales, one per 32) or
// kind::mxf4nvf4 (e4m3, one per 16), which multiplies e2m1 by e2m1, applies both scales and
// accumulates in float32.  The weights are the M side (128 rows per CTA, one TMEM lane each) and
// the tokens the N side, so one token costs an N = 32 tile and not a padded M.
//
// A pipeline stage holds 256 columns: the codes of 128 weight rows and the tile's token rows (128
// bytes a row, K-major, 128-byte swizzle) and their scale tiles (512 bytes per 128 rows x 4
// blocks), all by TMA.  The MMA warp copies each stage's scale tiles into tensor memory
// (tcgen05.cp 32x128b.warpx4; the operand's tile order is the order the MMA reads) and issues
// four MMAs of 64 columns.  tcgen05 copies and MMAs of one thread run in order, so the copy needs no
// wait, and the two scale buffers only keep the copy of one stage off the MMAs of the one before.
//
// Many tokens: SM pairs (cta_group::2) take 256 x 256 tiles.  Each CTA loads its 128 weight rows
// and half of the tokens, so an SM fetches 32 KB of codes per 256 columns where a one-SM 128 x 256
// tile fetches 48, and its tensor core reads two thirds of the shared memory: 8192 x 4096 ->
// 14336 (NVFP4) takes 258 us with one-SM tiles, 192 with pairs.  Both CTAs need the scales of all the tile's
// tokens.  The loads of both complete on the even CTA's barrier; its MMA warp issues for both.
//
// float32 results take the whole reduction in one chain of accumulations too, although each truncates: a product
// of two 4-bit values and their scales has few bits, so most additions are exact, and a chain has a quarter of the
// steps that it has with bf16.  Sums of positive products with block scales spread over 2^16 come out low
// by 2^-22 (4096 columns) to 2^-20 (14336) on average, which is what a float32 sum in another order is off by at
// its worst places.  Restarting every 16 MMAs made that 2^-22 for any length and cost 55 -> 149 us (2048 x 14336
// -> 4096): there is no room for a second accumulator, and the sums take all registers.
//
// The accumulator (256 columns) and the scales do not fit into tensor memory twice, so there is one
// accumulator: eight epilogue warps read it into registers at once and hand it back before they
// convert and store, while the next tile's MMAs run.
//
// Few tiles: a cluster of S CTAs splits the columns, each leaves its partial tile in its own
// shared memory, and after a cluster barrier each sums its share of the tile over the cluster in
// rank order (distributed shared memory: no workspace, no atomics, the same bits every run).
//
// Every wait is bounded (about a second); one that runs out sets the status word, stops the
// roles of the CTA (of both, in a pair), drains its loads and MMAs and frees its tensor memory.
#include "kquant_kernels.h"
#include "mx4_format.cuh"
#include "mx4_product.cuh"
#include "umma.cuh"

namespace cpk {
namespace {

__device__ int g_status;

constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;

template <int FMT, int NT, bool PAIR> struct Cfg {
  static constexpr int kAtoms = FMT == kMXFP4 ? 2 : 4;      // scale tiles per 128 rows x 256 columns
  static constexpr int kXT = NT > 128 ? 2 : 1;              // 128-row tiles of token scales
  static constexpr int kXRows = PAIR ? NT / 2 : NT;         // token rows this CTA loads
  static constexpr int kWBytes = 128 * 128, kXBytes = kXRows * 128;
  static constexpr int kSBytes = kAtoms * 512;              // scales of 128 rows
  static constexpr int kStage = kWBytes + kXBytes + (1 + kXT) * kSBytes;
  static constexpr int kFit = (224 * 1024) / kStage;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + 256;
  static constexpr int kScaleCols = (1 + kXT) * kAtoms * 4;   // TMEM columns of one stage's scales
  static constexpr int kCols = NT + 2 * kScaleCols;
  static constexpr uint32_t kTmem = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kStage % 1024 == 0, "stages keep the swizzle's alignment");
  // both operands e2m1 (bits 7-9, 10-11 = 1), K-major, N >> 3, scale type (1 = e8m0), M >> 4
  static constexpr uint32_t kIdesc = (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) |
                                     ((FMT == kMXFP4 ? 1u : 0u) << 23) | ((PAIR ? 16u : 8u) << 24);
};

struct MmParams {
  void* y;
  int64_t T, rows;
  float alpha;
  int dtype;
  int steps;            // 256-column steps
  int mtiles, tiles;    // weight tiles; weight tiles x token tiles
  Mx4Waits waits;
};

// Shared-memory descriptor of a scale tile for tcgen05.cp: no swizzle, 8 x 16-byte cores 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (8ull << 32) | (1ull << 46);
}
template <bool PAIR> __device__ __forceinline__ void scale_cp(uint32_t taddr, uint64_t desc) {
  if (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
#define CPK_UMMA_MX4(GROUP, KIND)                                                                        \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                        \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), \
               "l"(ad), "l"(bd), "r"(idesc), "r"(sa), "r"(sb), "r"(accum)                                \
               : "memory")
template <int FMT, bool PAIR>
__device__ __forceinline__ void umma_mx4(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sa, uint32_t sb,
                                         uint32_t accum) {
  if (FMT == kMXFP4) {
    if (PAIR) CPK_UMMA_MX4("2", "mxf4.block_scale.scale_vec::2X");
    else CPK_UMMA_MX4("1", "mxf4.block_scale.scale_vec::2X");
  } else {
    if (PAIR) CPK_UMMA_MX4("2", "mxf4nvf4.block_scale.scale_vec::4X");
    else CPK_UMMA_MX4("1", "mxf4nvf4.block_scale.scale_vec::4X");
  }
}
#undef CPK_UMMA_MX4

// PAIR: clusters of two CTAs share a 256-row tile, split = 1.  Else clusters of `split` CTAs share
// the columns of a 128-row tile.
template <int FMT, int NT, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    mx4_matmul_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                      const __grid_constant__ CUtensorMap map_sw, const __grid_constant__ CUtensorMap map_sx,
                      const MmParams prm, int split) {
  using C = Cfg<FMT, NT, PAIR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + C::kStages * C::kStage);   // full, empty, acc_full, acc_empty, done
  volatile int* misc = reinterpret_cast<volatile int*>(bars + 2 * C::kStages + 3);   // [0] tmem, [1] abort
  const uint32_t ring = smem_u32(base);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * C::kStages;
  const uint32_t accf = empty0 + 8 * C::kStages, acce = accf + 8, done = acce + 8;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = PAIR || split > 1 ? (int)cluster_rank() : 0;
  const bool leader = !PAIR || rank == 0;
  const int group = PAIR ? 2 : split;
  const int first = (int)blockIdx.x / group, stride = (int)gridDim.x / group;
  const int s_begin = PAIR ? 0 : (int)((int64_t)prm.steps * rank / split);
  const int s_end = PAIR ? prm.steps : (int)((int64_t)prm.steps * (rank + 1) / split);
  // first weight row of this CTA's part of a tile
  auto tile_row = [&](int tile) { return (int64_t)(tile % prm.mtiles) * (PAIR ? 256 : 128) + (PAIR ? rank * 128 : 0); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; s++) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(accf, 1);
    mbar_init(acce, PAIR ? 2 * kEpiWarps : kEpiWarps);
    mbar_init(done, 1);
    misc[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_sw)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_sx)) : "memory");
  }
  if (warp == 1) tmem_alloc<PAIR>(smem_u32((const void*)&misc[0]), C::kTmem);
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();   // both CTAs' barriers are initialised and their tensor memory allocated
  tc_fence_after();
  const uint32_t tmem = (uint32_t)misc[0];
  volatile int* abort = &misc[1];
  const uint32_t peer = PAIR ? rank ^ 1 : 0;
  const uint32_t peer_abort = PAIR ? peer_addr(smem_u32((const void*)&misc[1]), peer) : 0;
  auto fail = [&] {
    if (PAIR) fail_pair(abort, peer_abort, &g_status);
    else fail_cta(abort, &g_status);
  };

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t lead_full0 = PAIR ? peer_addr(full0, 0) : full0;
      const int groups = prm.steps * C::kAtoms;   // scale tiles per 128 rows
      int it = 0;
      bool ok = true;
      for (int tile = first; ok && tile < prm.tiles; tile += stride) {
        const int row = (int)tile_row(tile), t0 = tile / prm.mtiles * NT;
        for (int s = s_begin; s < s_end; s++, it++) {
          const int st = it % C::kStages, round = it / C::kStages;
          if (round > 0 && !mbar_wait(empty0 + 8 * st, (round - 1) & 1, abort, prm.waits.ns)) {
            ok = false;
            break;
          }
          if (it == prm.waits.skip) continue;
          const uint32_t fb = lead_full0 + 8 * st, sw = ring + st * C::kStage, sx = sw + C::kWBytes, ss = sx + C::kXBytes;
          // boxes past the arrays' ends arrive as zeros and count in full
          if (leader) mbar_expect_tx(full0 + 8 * st, (PAIR ? 2 : 1) * C::kStage);
          tma_load_group<PAIR>(sw, &map_w, s * 128, row, fb);
          tma_load_group<PAIR>(sx, &map_x, s * 128, t0 + (PAIR ? rank * C::kXRows : 0), fb);
          tma_load_group<PAIR>(ss, &map_sw, 0, row / 128 * groups + s * C::kAtoms, fb);
#pragma unroll
          for (int k = 0; k < C::kXT; k++)
            tma_load_group<PAIR>(ss + (1 + k) * C::kSBytes, &map_sx, 0, (t0 / 128 + k) * groups + s * C::kAtoms, fb);
        }
      }
      if (!ok) fail();
      // every load issued lands before the CTA goes on: the even CTA sees its full barriers, the
      // odd one the MMAs that consumed its loads (or the wait's bound)
      for (int k = max(0, it - C::kStages); k < it; k++) {
        int zero = 0;
        mbar_wait((leader ? full0 : empty0) + 8 * (k % C::kStages), (k / C::kStages) & 1, &zero, prm.waits.ns);
      }
    }
  } else if (warp == 1) {
    if (leader) {
      const bool elected = elect_one();
      int it = 0, n = 0;
      bool ok = true;
      for (int tile = first; ok && tile < prm.tiles; tile += stride, n++) {
        if (n > 0 && !mbar_wait_warp(acce, (n - 1) & 1, abort, prm.waits.ns)) {
          ok = false;
          break;
        }
        for (int s = s_begin; s < s_end; s++, it++) {
          const int st = it % C::kStages;
          if (!mbar_wait_warp(full0 + 8 * st, (it / C::kStages) & 1, abort, prm.waits.ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sw = ring + st * C::kStage, sx = sw + C::kWBytes;
          const uint64_t ad = sw128_desc(sw, 16, 1024), bd = sw128_desc(sx, 16, 1024), sd = scale_desc(sx + C::kXBytes);
          const uint32_t ta = tmem + NT + (it & 1) * C::kScaleCols, tb = ta + C::kAtoms * 4;
          const uint32_t more = s > s_begin;
          if (elected) {   // descriptors count in 16 bytes
#pragma unroll
            for (int a = 0; a < C::kAtoms; a++) {
              scale_cp<PAIR>(ta + 4 * a, sd + a * 32);
#pragma unroll
              for (int k = 0; k < C::kXT; k++)
                scale_cp<PAIR>(tb + (a * C::kXT + k) * 4, sd + (1 + k) * (C::kSBytes / 16) + a * 32);
            }
#pragma unroll
            for (int kk = 0; kk < 4; kk++) {
              const int atom = FMT == kMXFP4 ? kk / 2 : kk;
              const uint32_t id = FMT == kMXFP4 ? (kk & 1) * 2u : 0u;   // which half of the scale word
              umma_mx4<FMT, PAIR>(tmem, ad + 2 * kk, bd + 2 * kk, C::kIdesc | (id << 4) | (id << 29), ta + 4 * atom,
                                  tb + 4 * C::kXT * atom, kk > 0 ? 1u : more);
            }
            umma_commit_group<PAIR>(empty0 + 8 * st);
          }
          __syncwarp();
        }
        if (ok && elected) umma_commit_group<PAIR>(accf);
        __syncwarp();
      }
      if (!ok) fail();
      // all MMAs complete before tensor memory is freed and before the other CTA may exit
      if (elected) umma_commit_group<PAIR>(done);
      int zero = 0;
      mbar_wait(done, 0, &zero, prm.waits.ns);
    }
  } else {
    const int q = warp & 3, hh = (warp - 2) >> 2;
    const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16) + hh * (NT / 2);
    const uint32_t lead_acce = PAIR ? peer_addr(acce, 0) : acce;
    int n = 0;
    for (int tile = first; tile < prm.tiles; tile += stride, n++) {
      if (!mbar_wait_warp(accf, n & 1, abort, prm.waits.ns)) {
        fail();
        break;
      }
      tc_fence_after();
      float v[NT / 2];
      tmem_ld_cols(trow, v);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader) mbar_arrive(acce);
        else mbar_arrive_remote(lead_acce);
      }
      if (split > 1) {   // the loads and MMAs of this CTA's only tile are complete: the ring is free
        float* part = reinterpret_cast<float*>(base);
#pragma unroll
        for (int c = 0; c < NT / 2; c++) part[(hh * (NT / 2) + c) * 128 + 32 * q + lane] = v[c];
      } else {
        store_tile<NT / 2>(v, prm.alpha, prm.y, prm.dtype, tile_row(tile) + 32 * q, prm.rows,
                           (int64_t)(tile / prm.mtiles) * NT + hh * (NT / 2), prm.T);
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (PAIR) {
    cluster_sync();   // neither CTA touches the other's memory from here on
  } else if (split > 1) {
    cluster_sync();
    const int64_t t0 = (int64_t)(first / prm.mtiles) * NT;
    join_partials(base, rank, split, (int)min((int64_t)NT, prm.T - t0), tile_row(first), t0, prm.rows, prm.alpha,
                  prm.dtype, prm.y);
    cluster_sync();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_free<PAIR>(tmem, C::kTmem);
  }
}

template <int FMT, int NT, bool PAIR>
int launch_tiles(const Mx4View& a, const Mx4View& w, float alpha, int dtype, void* y, int split, cudaStream_t stream) {
  using C = Cfg<FMT, NT, PAIR>;
  CUtensorMap mw, mx, msw, msx;
  const int64_t pitch = mx4_pitch(w.n), steps = pitch / 128;
  const int64_t wt = (w.rows + 127) / 128, xt = (a.rows + 127) / 128;
  if (!codes_map(&mw, w.codes, pitch, w.rows, 128, 128) || !codes_map(&mx, a.codes, pitch, a.rows, 128, C::kXRows) ||
      !scales_map(&msw, w.scales, wt * steps * C::kAtoms, C::kAtoms) ||
      !scales_map(&msx, a.scales, xt * steps * C::kAtoms, C::kAtoms))
    return 5;
  MmParams p;
  p.y = y;
  p.T = a.rows;
  p.rows = w.rows;
  p.alpha = alpha;
  p.dtype = dtype;
  p.steps = (int)steps;
  p.mtiles = (int)(PAIR ? (wt + 1) / 2 : wt);
  p.tiles = p.mtiles * (int)((a.rows + NT - 1) / NT);
  p.waits = mx4_take_waits();
  const int sms = device_sm_count();
  const int grid = PAIR ? 2 * std::min(p.tiles, sms / 2) : split > 1 ? p.tiles * split : std::min(p.tiles, sms);
  return launch_cluster<mx4_matmul_kernel<FMT, NT, PAIR>>(grid, kThreads, C::kSmem, PAIR ? 2 : split, stream, mw, mx, msw,
                                                         msx, p, split);
}

template <int FMT>
int launch_format(const Mx4View& a, const Mx4View& w, float alpha, int dtype, void* y, cudaStream_t stream) {
  const int sms = device_sm_count();
  const int64_t mt = (w.rows + 127) / 128, T = a.rows;
  const int steps = (int)(mx4_pitch(w.n) / 128);
  const int nt = T <= 32 ? 32 : T <= 64 ? 64 : 128;
  const int64_t tiles = mt * ((T + nt - 1) / nt);
  const int64_t pairs = (mt + 1) / 2 * ((T + 255) / 256);
  // 256-column steps take about 600 clocks in a one-SM tile, and in a pair's, of four times the work, 700
  double one;
  const int split = best_split(tiles, steps, 600, nt, sms, &one);
  if (T > 128 && (double)((pairs + sms / 2 - 1) / (sms / 2)) * steps * 700 + 3500 <= one)
    return launch_tiles<FMT, 256, true>(a, w, alpha, dtype, y, 1, stream);
  switch (nt) {
    case 32: return launch_tiles<FMT, 32, false>(a, w, alpha, dtype, y, split, stream);
    case 64: return launch_tiles<FMT, 64, false>(a, w, alpha, dtype, y, split, stream);
    default: return launch_tiles<FMT, 128, false>(a, w, alpha, dtype, y, split, stream);
  }
}

}  // namespace

int launch_mx4_matmul(const Mx4View& a, const Mx4View& w, float alpha, int dtype, void* y, cudaStream_t stream) {
  if (!bind_context()) return 6;
  return w.fmt == kMXFP4 ? launch_format<kMXFP4>(a, w, alpha, dtype, y, stream)
                         : launch_format<kNVFP4>(a, w, alpha, dtype, y, stream);
}

int mx4_matmul_status(cudaStream_t stream, int* status) { return read_status_word(g_status, stream, status); }

}  // namespace cpk
