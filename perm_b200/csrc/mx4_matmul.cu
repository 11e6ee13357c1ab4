// y = alpha * a w^T for two 4-bit operands of one format: a [T, n] (tokens), w [rows, n] (weights).
//
// Block-scaled tensor-core kernel: tcgen05.mma kind::mxf4 (e8m0 scales, one per 32) or
// kind::mxf4nvf4 (e4m3, one per 16), which multiplies e2m1 by e2m1, applies both scales and
// accumulates in float32.  The weights are the M side (128 rows per CTA, one TMEM lane each) and
// the tokens the N side, so one token costs an N = 32 tile and not a padded M.
//
// A pipeline stage holds 256 columns: the codes of 128 weight rows and NT token rows (128 bytes a
// row, K-major, 128-byte swizzle, by TMA) and their scale tiles (512 bytes per 128 rows x 4
// blocks, by plain bulk copies).  The MMA thread copies each stage's scale tiles into tensor memory
// (tcgen05.cp 32x128b.warpx4; the operand's tile order is the order the MMA reads) and issues
// four MMAs of 64 columns.  tcgen05 copies and MMAs of one thread run in order, so the copy needs no
// wait, and the two scale buffers only keep the copy of one stage off the MMAs of the one before.
//
// The accumulator (NT columns) and the scales do not fit twice at NT = 256, so there is one
// accumulator: eight epilogue warps read it into registers at once and hand it back before they
// convert and store, while the next tile's MMAs run.
//
// Few tiles: a cluster of S CTAs splits the columns, each leaves its partial tile in its own
// shared memory, and after a cluster barrier each sums its share of the tile over the cluster in
// rank order (distributed shared memory: no workspace, no atomics, the same bits every run).
//
// Every wait is bounded (about a second); one that runs out sets the status word, stops the
// CTA's roles, drains its loads and MMAs and frees its tensor memory.
#include "kquant_kernels.h"
#include "mx4_format.cuh"
#include "mx4_product.cuh"
#include "umma.cuh"

namespace cpk {
namespace {

__device__ int g_status;

constexpr unsigned long long kWaitNs = 1000000000ull;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;

template <int FMT, int NT> struct Cfg {
  static constexpr int kAtoms = FMT == kMXFP4 ? 2 : 4;      // scale tiles per 128 rows x 256 columns
  static constexpr int kXT = NT > 128 ? 2 : 1;              // 128-row tiles of token scales
  static constexpr int kWBytes = 128 * 128, kXBytes = NT * 128;
  static constexpr int kSBytes = kAtoms * 512;              // scales of 128 rows
  static constexpr int kStage = kWBytes + kXBytes + (1 + kXT) * kSBytes;
  static constexpr int kFit = (224 * 1024) / kStage;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + 256;
  static constexpr int kScaleCols = (1 + kXT) * kAtoms * 4;   // TMEM columns of one stage's scales
  static constexpr int kCols = NT + 2 * kScaleCols;
  static constexpr uint32_t kTmem = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kStage % 1024 == 0, "stages keep the swizzle's alignment");
  // both operands e2m1 (bits 7-9, 10-11 = 1), K-major, N >> 3, scale type (1 = e8m0), M = 128
  static constexpr uint32_t kIdesc = (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) |
                                     ((FMT == kMXFP4 ? 1u : 0u) << 23) | (8u << 24);
};

struct MmParams {
  const uint8_t* w_scales;
  const uint8_t* x_scales;
  void* y;
  int64_t T, rows;
  float alpha;
  int dtype;
  int steps;            // 256-column steps
  int mtiles, tiles;    // weight tiles; weight tiles x token tiles
  int xtiles;           // 128-row tiles of the tokens' scales
};

// Shared-memory descriptor of a scale tile for tcgen05.cp: no swizzle, 8 x 16-byte cores 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (8ull << 32) | (1ull << 46);
}
__device__ __forceinline__ void scale_cp(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int FMT>
__device__ __forceinline__ void umma_mx4(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sa, uint32_t sb,
                                         uint32_t accum) {
  if (FMT == kMXFP4)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(sa), "r"(sb), "r"(accum)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(sa), "r"(sb), "r"(accum)
        : "memory");
}

template <int FMT, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    mx4_matmul_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                      const MmParams prm, int split) {
  using C = Cfg<FMT, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + C::kStages * C::kStage);   // full, empty, acc_full, acc_empty, done
  volatile int* misc = reinterpret_cast<volatile int*>(bars + 2 * C::kStages + 3);   // [0] tmem, [1] abort
  const uint32_t ring = smem_u32(base);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * C::kStages;
  const uint32_t accf = empty0 + 8 * C::kStages, acce = accf + 8, done = acce + 8;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int first = (int)blockIdx.x / split, stride = (int)gridDim.x / split;
  const int s_begin = (int)((int64_t)prm.steps * rank / split), s_end = (int)((int64_t)prm.steps * (rank + 1) / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; s++) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(accf, 1);
    mbar_init(acce, kEpiWarps);
    mbar_init(done, 1);
    misc[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)&misc[0])),
                 "r"(C::kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)misc[0];
  volatile int* abort = &misc[1];

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int tile = first; ok && tile < prm.tiles; tile += stride) {
        const int m = tile % prm.mtiles, t = tile / prm.mtiles;
        const int xt = t * NT / 128, nx = min(C::kXT, prm.xtiles - xt);   // token scale tiles that exist
        for (int s = s_begin; s < s_end; s++, it++) {
          const int st = it % C::kStages, round = it / C::kStages;
          if (round > 0 && !mbar_wait(empty0 + 8 * st, (round - 1) & 1, abort, kWaitNs)) {
            ok = false;
            break;
          }
          const uint32_t fb = full0 + 8 * st, sw = ring + st * C::kStage, sx = sw + C::kWBytes, ss = sx + C::kXBytes;
          mbar_expect_tx(fb, C::kWBytes + C::kXBytes + (1 + nx) * C::kSBytes);
          tma_load(sw, &map_w, s * 128, m * 128, fb);
          tma_load(sx, &map_x, s * 128, t * NT, fb);
          const int64_t per = (int64_t)prm.steps * C::kSBytes;   // scale bytes of 128 rows
          bulk_load(ss, prm.w_scales + m * per + (int64_t)s * C::kSBytes, C::kSBytes, fb);
          for (int k = 0; k < nx; k++)
            bulk_load(ss + (1 + k) * C::kSBytes, prm.x_scales + (xt + k) * per + (int64_t)s * C::kSBytes, C::kSBytes, fb);
        }
      }
      if (!ok) fail_cta(abort, &g_status);
      // every load issued lands before the CTA goes on
      for (int k = max(0, it - C::kStages); k < it; k++) {
        int zero = 0;
        mbar_wait(full0 + 8 * (k % C::kStages), (k / C::kStages) & 1, &zero, kWaitNs);
      }
    }
  } else if (warp == 1) {
    const bool elected = elect_one();
    int it = 0, n = 0;
    bool ok = true;
    for (int tile = first; ok && tile < prm.tiles; tile += stride, n++) {
      if (n > 0 && !mbar_wait_warp(acce, (n - 1) & 1, abort, kWaitNs)) {
        ok = false;
        break;
      }
      for (int s = s_begin; s < s_end; s++, it++) {
        const int st = it % C::kStages;
        if (!mbar_wait_warp(full0 + 8 * st, (it / C::kStages) & 1, abort, kWaitNs)) {
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
            scale_cp(ta + 4 * a, sd + a * 32);
#pragma unroll
            for (int k = 0; k < C::kXT; k++) scale_cp(tb + (a * C::kXT + k) * 4, sd + (1 + k) * (C::kSBytes / 16) + a * 32);
          }
#pragma unroll
          for (int kk = 0; kk < 4; kk++) {
            const int atom = FMT == kMXFP4 ? kk / 2 : kk;
            const uint32_t id = FMT == kMXFP4 ? (kk & 1) * 2u : 0u;   // which half of the scale word
            umma_mx4<FMT>(tmem, ad + 2 * kk, bd + 2 * kk, C::kIdesc | (id << 4) | (id << 29), ta + 4 * atom,
                          tb + 4 * C::kXT * atom, kk > 0 ? 1u : more);
          }
          umma_commit(empty0 + 8 * st);
        }
        __syncwarp();
      }
      if (ok && elected) umma_commit(accf);
      __syncwarp();
    }
    if (!ok) fail_cta(abort, &g_status);
    if (elected) umma_commit(done);   // all MMAs complete before tensor memory is freed
    int zero = 0;
    mbar_wait(done, 0, &zero, kWaitNs);
  } else {
    const int q = warp & 3, hh = (warp - 2) >> 2;
    const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16) + hh * (NT / 2);
    int n = 0;
    for (int tile = first; tile < prm.tiles; tile += stride, n++) {
      const bool got = mbar_wait(accf, n & 1, abort, kWaitNs);
      if (!__all_sync(0xffffffffu, got)) {
        fail_cta(abort, &g_status);
        break;
      }
      tc_fence_after();
      float v[NT / 2];
#pragma unroll
      for (int c = 0; c < NT / 2; c += 16) tmem_ld16(trow + c, *reinterpret_cast<float(*)[16]>(v + c));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acce);
      const int r = 32 * q + lane;
      if (split > 1) {   // the loads and MMAs of this CTA's only tile are complete: the ring is free
        float* part = reinterpret_cast<float*>(base);
#pragma unroll
        for (int c = 0; c < NT / 2; c++) part[(hh * (NT / 2) + c) * 128 + r] = v[c];
      } else {
        store_tile<NT / 2>(v, prm.alpha, prm.y, prm.dtype, (int64_t)(tile % prm.mtiles) * 128 + 32 * q, prm.rows,
                           (int64_t)(tile / prm.mtiles) * NT + hh * (NT / 2), prm.T);
      }
    }
  }
  __syncwarp();
  if (split > 1) {
    cluster_sync();
    const int64_t row0 = (int64_t)(first % prm.mtiles) * 128, t0 = (int64_t)(first / prm.mtiles) * NT;
    const int cols = (int)min((int64_t)NT, prm.T - t0);
    join_partials(base, rank, split, cols, row0, t0, prm.rows, prm.alpha, prm.dtype, prm.y);
    cluster_sync();
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem) : "memory");
  }
}

template <int FMT, int NT>
int launch_tiles(const Mx4View& a, const Mx4View& w, float alpha, int dtype, void* y, int split, cudaStream_t stream) {
  using C = Cfg<FMT, NT>;
  CUtensorMap mw, mx;
  const int64_t pitch = mx4_pitch(w.n);
  if (!codes_map(&mw, w.codes, pitch, w.rows, 128, 128) || !codes_map(&mx, a.codes, pitch, a.rows, 128, NT)) return 5;
  MmParams p;
  p.w_scales = w.scales;
  p.x_scales = a.scales;
  p.y = y;
  p.T = a.rows;
  p.rows = w.rows;
  p.alpha = alpha;
  p.dtype = dtype;
  p.steps = (int)(pitch / 128);
  p.mtiles = (int)((w.rows + 127) / 128);
  p.tiles = p.mtiles * (int)((a.rows + NT - 1) / NT);
  p.xtiles = (int)((a.rows + 127) / 128);
  const int grid = split > 1 ? p.tiles * split : std::min(p.tiles, device_sm_count());
  return launch_cluster<mx4_matmul_kernel<FMT, NT>>(grid, kThreads, C::kSmem, split, stream, mw, mx, p, split);
}

template <int FMT>
int launch_format(const Mx4View& a, const Mx4View& w, float alpha, int dtype, void* y, cudaStream_t stream) {
  const int sms = device_sm_count();
  const int64_t mt = (w.rows + 127) / 128, T = a.rows;
  const int steps = (int)(mx4_pitch(w.n) / 128);
  auto tiles = [&](int nt) { return mt * ((T + nt - 1) / nt); };
  int nt = T <= 32 ? 32 : T <= 64 ? 64 : 128;
  // a 256-token tile halves the weights' traffic per product, but needs enough tiles to fill the SMs
  if (T > 128 && (tiles(256) + sms - 1) / sms * 2 <= (tiles(128) + sms - 1) / sms) nt = 256;
  int split = 1;
  if (nt <= 128)
    while (split < 8 && tiles(nt) * split * 2 <= sms && split * 2 <= steps) split *= 2;
  switch (nt) {
    case 32: return launch_tiles<FMT, 32>(a, w, alpha, dtype, y, split, stream);
    case 64: return launch_tiles<FMT, 64>(a, w, alpha, dtype, y, split, stream);
    case 128: return launch_tiles<FMT, 128>(a, w, alpha, dtype, y, split, stream);
    default: return launch_tiles<FMT, 256>(a, w, alpha, dtype, y, split, stream);
  }
}

}  // namespace

int launch_mx4_matmul(const Mx4View& a, const Mx4View& w, float alpha, int dtype, void* y, cudaStream_t stream) {
  return w.fmt == kMXFP4 ? launch_format<kMXFP4>(a, w, alpha, dtype, y, stream)
                         : launch_format<kNVFP4>(a, w, alpha, dtype, y, stream);
}

int mx4_matmul_status(cudaStream_t stream, int* status) { return read_status_word(g_status, stream, status); }

}  // namespace cpk
