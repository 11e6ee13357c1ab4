// Products of activations in their own type with frozen 4-bit weights w [rows, n]:
//   y = alpha * x w^T   (x [T, n], TR = false)
//   y = alpha * x w     (x [T, rows], TR = true: the first form's gradient with respect to x)
//
// Tensor-core kernel (tcgen05 kind::f16, bf16 x bf16 -> f32).  An e2m1 value times its block scale
// has at most six significant bits, so it is exact in bf16, and so is every product in the float32
// accumulator.  The 4-bit weights go from global to shared memory as they are (TMA), 128 x 128 at a
// time, and decoding warps write them as the swizzled bf16 tile that the MMA reads: K-major for
// x w^T, MN-major for x w, where the packed axis is the output's.  Both are the same bytes: two
// halves of 64 columns, 128 bytes a row.  Weights are the M side (128 rows of the output per CTA), tokens the N side.
//
// Decoding.  A conversion turns two codes into two f16 values; widened to float32 they take the block
// scale, exactly, and go back as a pair of bf16.  (Shifting the f16 bits into a bf16 with another exponent
// and one bf16 product takes an instruction less, but three of its five are for the pipe that the
// conversions use too: 4 to 10 % slower.)
//
// float16 and float32 activations are cut into bf16 parts (8 significant bits each: two for float16,
// three for float32, no remainder) by a first kernel, and every decoded weight tile is multiplied
// by all the parts, so the result is that of the activations as they are.  Rows of x that TMA
// cannot address (not 16-byte aligned) go through the same kernel.
//
// Work split, joins and bounded waits are those of the 4-bit products: SM pairs on 256 x 256 tiles
// for many tokens, clusters over the reduction where there are few tiles (mx4_matmul.cu).  Two
// accumulators alternate, so storing one tile overlaps the MMAs of the next.  float32 results restart the
// accumulation every step (24 MMAs, the smallest part of x first) and sum the chunks in round-to-nearest
// registers, because the tensor core's own accumulation truncates: sums of positive products come out low by 2^-24 on
// average (2^-19 with the largest part first, which has the other parts' MMAs truncate the whole sum too).
#include "mx4_dense.cuh"
#include "mx4_product.cuh"

namespace cpk {
namespace {

__device__ int g_status;

constexpr int kChunkSteps = 1;  // 128-deep steps of one float32 accumulation chain

template <int FMT, int NT, bool PAIR, bool TR, bool CHUNK> struct Cfg {
  // warps: 0 x loads, 1 MMA, 2 code loads, 3 allocation, 4-7 epilogue, then groups of eight that decode
  // steps in turn.  float32 results keep NT sums per epilogue thread, which leaves registers for one group.
  // A pair has the registers for a third group (MXFP4, bf16, 4096 -> 14336: 512 tokens 78 us with
  // two, 62 with three, 4096 tokens 474 and 420); one-SM tiles were no faster with it.
  static constexpr int kGroups = CHUNK ? 1 : PAIR ? 3 : 2;
  static constexpr int kThreads = 256 + 256 * kGroups;
  static constexpr int kXRows = PAIR ? NT / 2 : NT;
  static constexpr int kA = 128 * 256;                     // decoded tile: 128 rows x 128, bf16
  static constexpr int kB = kXRows * 256;                  // tokens x 128, bf16
  static constexpr int kAtoms = FMT == kMXFP4 ? 1 : 2;     // scale tiles of 128 x 128 codes
  static constexpr int kCodes = 128 * 64;
  static constexpr int kC = (kCodes + kAtoms * 512 + 1023) / 1024 * 1024;
  // code stages at most; see LinParams::turns
  static constexpr int kCS = PAIR ? 3 : 2, kMaxStages = 6;
  static constexpr int kRing = (225 * 1024 - kCS * kC) / 1024 * 1024;   // stages of one decoded tile and its x tiles
  static constexpr size_t kSmem = 1024 + (size_t)kRing + kCS * kC + 512;
  static constexpr uint32_t kTmem = 2 * NT < 64 ? 64 : 2 * NT;
  static_assert(kCS % kGroups == 0, "code stages for every group");
  static_assert(kB % 1024 == 0 && kRing >= NT * 512, "stages keep the swizzle's alignment, and a partial tile fits");
  // f32 accumulator, A and B bf16, A MN-major in the transposed form, N >> 3, M >> 4
  static constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((TR ? 1u : 0u) << 15) |
                                     ((uint32_t)(NT >> 3) << 17) | ((PAIR ? 16u : 8u) << 24);
};

struct LinParams {
  void* y;
  int64_t T, out;       // y is [T, out]
  int64_t wrows;        // rows of w
  float alpha;
  int dtype;
  int parts;
  int nst;              // stages of the ring
  // The groups that decode, and the code stages.  A wait for a phase of a barrier is answered by its parity, so it
  // must not come before the phase ahead of the one meant is known to be over.  The ring's stages: a group that
  // decodes step s waits for the MMAs of s - nst, and has seen those of s - turns - nst complete; the phase
  // ahead is that of s - 2 nst, so turns <= nst.  The code stages: their number is a multiple of turns,
  // so that one group sees every use of a stage.
  int turns, ncs;
  int steps;            // 128-deep steps of the reduction
  int groups;           // scale tiles per 128 rows of w
  int mtiles, tiles;
  Mx4Waits waits;
};

// Eight codes times a block scale -> eight bf16 values in pairs.
__device__ __forceinline__ void decode8(uint32_t w, float scale, uint32_t (&v)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __fmul2_rn(__half22float2(*reinterpret_cast<const __half2*>(&v[i])), make_float2(scale, scale));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v[i]) : "f"(f.y), "f"(f.x));
  }
}

template <int FMT, int NT, bool PAIR, bool TR, bool CHUNK>
__global__ void __launch_bounds__((Cfg<FMT, NT, PAIR, TR, CHUNK>::kThreads), 1)
    mx4_linear_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_s,
                      const __grid_constant__ CUtensorMap map_x, const LinParams prm, int split) {
  using C = Cfg<FMT, NT, PAIR, TR, CHUNK>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + C::kRing + C::kCS * C::kC);
  constexpr int kBars = 2 * (C::kMaxStages + C::kCS) + 5;
  volatile int* misc = reinterpret_cast<volatile int*>(bars + kBars);   // [0] tmem, [1] abort
  const int nst = prm.nst, stage_bytes = C::kA + prm.parts * C::kB;
  const uint32_t ring = smem_u32(base), ring_c = ring + C::kRing;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * C::kMaxStages;
  const uint32_t cfull = empty0 + 8 * C::kMaxStages, cempty = cfull + 8 * C::kCS;
  const uint32_t accf = cempty + 8 * C::kCS, acce = accf + 16, done = acce + 16;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = PAIR || split > 1 ? (int)cluster_rank() : 0;
  const bool leader = !PAIR || rank == 0;
  const int group = PAIR ? 2 : split;
  const int first = (int)blockIdx.x / group, stride = (int)gridDim.x / group;
  const int s_begin = PAIR ? 0 : (int)((int64_t)prm.steps * rank / split);   // this CTA's steps
  const int s_end = PAIR ? prm.steps : (int)((int64_t)prm.steps * (rank + 1) / split);
  auto tile_row = [&](int tile) { return (int64_t)(tile % prm.mtiles) * (PAIR ? 256 : 128) + (PAIR ? rank * 128 : 0); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kMaxStages; s++) {
      mbar_init(full0 + 8 * s, 1 + (PAIR ? 16 : 8));   // the x loads, and the warps that decode the step
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int s = 0; s < C::kCS; s++) {
      mbar_init(cfull + 8 * s, 1);
      mbar_init(cempty + 8 * s, 8);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(accf + 8 * b, 1);
      mbar_init(acce + 8 * b, PAIR ? 8 : 4);
    }
    mbar_init(done, 1);
    misc[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_s)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
  }
  if (warp == 3) tmem_alloc<PAIR>(smem_u32((const void*)&misc[0]), C::kTmem);
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();   // both CTAs' barriers are initialised and their tensor memory allocated
  tc_fence_after();
  const uint32_t tmem = (uint32_t)misc[0];
  volatile int* abort = &misc[1];
  const uint32_t peer_abort = PAIR ? peer_addr(smem_u32((const void*)&misc[1]), rank ^ 1) : 0;
  auto fail = [&] {
    if (PAIR) fail_pair(abort, peer_abort, &g_status);
    else fail_cta(abort, &g_status);
  };

  if (warp == 0) {
    if (lane == 0) {   // ---- x tiles, all parts of a step
      const uint32_t lead_full = PAIR ? peer_addr(full0, 0) : full0;
      Ring rg{0, 0};
      int loads = 0;
      bool ok = true;
      for (int tile = first; ok && tile < prm.tiles; tile += stride) {
        const int t0 = tile / prm.mtiles * NT + (PAIR ? rank * C::kXRows : 0);
        for (int s = s_begin; s < s_end; s++, loads++) {
          if (loads >= nst && !mbar_wait(empty0 + 8 * rg.st, rg.ph ^ 1, abort, prm.waits.ns)) {
            ok = false;
            break;
          }
          if (loads != prm.waits.skip) {
            if (leader) mbar_expect_tx(full0 + 8 * rg.st, (PAIR ? 2 : 1) * prm.parts * C::kB);
            const uint32_t sx = ring + rg.st * stage_bytes + C::kA;
            for (int p = 0; p < prm.parts; p++)
#pragma unroll
              for (int k = 0; k < 2; k++)
                tma_load_group<PAIR>(sx + p * C::kB + k * (C::kB / 2), &map_x, s * 128 + k * 64, (int)(p * prm.T) + t0,
                                     lead_full + 8 * rg.st);
          }
          rg.advance(nst);
        }
      }
      if (!ok) fail();
      // Every load issued lands before the CTA goes on.  With all roles well, the last stages' MMAs,
      // which waited for them, show that; after a failure the decoders may be missing from the
      // full barriers, so wait as long as a load could take.
      for (int k = min(loads, nst); ok && k > 0; k--) {
        rg.back(nst);
        ok = mbar_wait(empty0 + 8 * rg.st, rg.ph, abort, prm.waits.ns);
      }
      if (!ok) {
        const unsigned long long t0 = gtime();
        while (gtime() - t0 < 2000000ull) __nanosleep(10000);
      }
    }
  } else if (warp == 2) {
    if (lane == 0) {   // ---- codes and scales of this CTA's rows
      Ring rc{0, 0};
      int it = 0;
      bool ok = true;
      for (int tile = first; ok && tile < prm.tiles; tile += stride) {
        const int m0 = (int)tile_row(tile);
        for (int s = s_begin; s < s_end; s++, it++, rc.advance(prm.ncs)) {
          const int st = rc.st;
          if (it >= prm.ncs && !mbar_wait(cempty + 8 * st, rc.ph ^ 1, abort, prm.waits.ns)) {
            ok = false;
            break;
          }
          const uint32_t fb = cfull + 8 * st, sc = ring_c + st * C::kC;
          mbar_expect_tx(fb, C::kCodes + C::kAtoms * 512);
          if (TR) {
            tma_load(sc, &map_w, m0 / 2, s * 128, fb);
            tma_load(sc + C::kCodes, &map_s, 0, s * prm.groups + m0 / 128 * C::kAtoms, fb);
          } else {
            tma_load(sc, &map_w, s * 64, m0, fb);
            tma_load(sc + C::kCodes, &map_s, 0, m0 / 128 * prm.groups + s * C::kAtoms, fb);
          }
        }
      }
      if (!ok) fail();
      for (int k = min(it, prm.ncs); k > 0; k--) {
        int zero = 0;
        rc.back(prm.ncs);
        mbar_wait(cfull + 8 * rc.st, rc.ph, &zero, prm.waits.ns);
      }
    }
  } else if (warp == 1) {
    if (leader) {   // ---- MMAs
      const bool elected = elect_one();
      Ring rg{0, 0};
      int cg = 0;
      bool ok = true;
      for (int tile = first; ok && tile < prm.tiles; tile += stride) {
        for (int g0 = s_begin; ok && g0 < s_end; cg++) {
          const int b = cg & 1, g1 = CHUNK ? min(s_end, g0 + kChunkSteps) : s_end;
          const uint32_t acc = tmem + b * NT;
          if (cg >= 2 && !mbar_wait_warp(acce + 8 * b, ((cg >> 1) - 1) & 1, abort, prm.waits.ns)) {
            ok = false;
            break;
          }
          for (int s = g0; s < g1; s++) {
            if (!mbar_wait_warp<PAIR>(full0 + 8 * rg.st, rg.ph, abort, prm.waits.ns)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = ring + rg.st * stage_bytes;
            const uint64_t ad = TR ? sw128_desc(sa, 16384, 1024) : sw128_desc(sa, 16, 1024);
            const uint64_t bd = sw128_desc(sa + C::kA, 16, 1024);
            if (elected) {
              for (int p = prm.parts - 1; p >= 0; p--)   // the smallest part first: what truncation takes goes by the sum
#pragma unroll
                for (int kk = 0; kk < 8; kk++)   // 16 deep: 32 bytes of a K-major row (four to a half), or 16 rows
                  umma_bf16<PAIR>(acc, ad + (TR ? 128 * kk : kk / 4 * 1024 + kk % 4 * 2),
                                  bd + p * (C::kB / 16) + kk / 4 * (C::kB / 32) + kk % 4 * 2, C::kIdesc,
                                  (uint32_t)(s - g0) | (p ^ (prm.parts - 1)) | kk);
              umma_commit_group<PAIR>(empty0 + 8 * rg.st);
            }
            __syncwarp();
            rg.advance(nst);
          }
          if (ok && elected) umma_commit_group<PAIR>(accf + 8 * b);
          __syncwarp();
          g0 = g1;
        }
      }
      if (!ok) fail();
      if (elected) umma_commit_group<PAIR>(done);   // all MMAs complete before tensor memory is freed
      int zero = 0;
      mbar_wait(done, 0, &zero, prm.waits.ns);
    }
  } else if (warp >= 8) {
    // ---- decoding.  Groups take steps in turn, so one group's waits and fences overlap the others' work; a
    // thread takes 64 codes (32 bytes): half of a row's 128.  It decodes into registers before it waits for the
    // stage.
    const int d = threadIdx.x & 255, g = (threadIdx.x - 256) >> 8;
    const int r = d & 127, h = d >> 7, x7 = r & 7;
    const uint32_t dst0 = h * 16384 + r * 128;
    const uint32_t at0 = r * 64 + (((h * 2) ^ ((r >> 1) & 3)) << 4), at1 = r * 64 + (((h * 2 + 1) ^ ((r >> 1) & 3)) << 4);
    const int srow = (r & 31) * 16 + (r >> 5) * 4;
    const uint32_t lead_full = PAIR ? peer_addr(full0, 0) : full0;
    Ring rg{0, 0}, rc{0, 0}, turn{0, 0};
    int seen = 0;
    bool ok = true;
    for (int tile = g < prm.turns ? first : prm.tiles; ok && tile < prm.tiles; tile += stride)
      for (int s = s_begin; s < s_end; s++, seen++, rg.advance(nst), rc.advance(prm.ncs), turn.advance(prm.turns)) {
        if (turn.st != g) continue;
        const int cs = rc.st;
        if (!mbar_wait_warp(cfull + 8 * cs, rc.ph, abort, prm.waits.ns)) {
          ok = false;
          break;
        }
        const uint32_t codes = ring_c + cs * C::kC, scales = codes + C::kCodes + srow;
        {
          const uint4 q[2] = {ld_stage_u32x4(codes + at0), ld_stage_u32x4(codes + at1)};
          float f[4];
          if (FMT == kMXFP4) {
            const uint32_t two = ld_stage_u16(scales + h * 2);
            f[0] = f[1] = e8m0_value(two & 0xFF);
            f[2] = f[3] = e8m0_value(two >> 8);
          } else {
            const uint32_t four = ld_stage_u32(scales + h * 512);
#pragma unroll
            for (int j = 0; j < 4; j++) f[j] = e4m3_value((four >> (8 * j)) & 0xFF);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(cempty + 8 * cs);   // the stage's bytes are in registers
          // rows past the last (their scale bytes are not defined) are part of the reduction: zero
          if (TR && (int64_t)s * 128 + r >= prm.wrows) f[0] = f[1] = f[2] = f[3] = 0.0f;
          uint32_t v[8][4];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const uint4& qq = q[i / 4];
            decode8(i % 4 == 0 ? qq.x : i % 4 == 1 ? qq.y : i % 4 == 2 ? qq.z : qq.w, f[i / 2], v[i]);
          }
          if (seen >= nst && !mbar_wait_warp(empty0 + 8 * rg.st, rg.ph ^ 1, abort, prm.waits.ns)) {
            ok = false;
            break;
          }
          const uint32_t dst = ring + rg.st * stage_bytes + dst0;
#pragma unroll
          for (int i = 0; i < 8; i++)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + ((i ^ x7) << 4)), "r"(v[i][0]), "r"(v[i][1]),
                         "r"(v[i][2]), "r"(v[i][3])
                         : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the MMAs read through the async proxy
        __syncwarp();
        if (lane == 0) {
          if (leader) mbar_arrive(full0 + 8 * rg.st);
          else mbar_arrive_remote_release(lead_full + 8 * rg.st);
        }
      }
    if (!ok) fail();
  } else if (warp >= 4) {
    // ---- epilogue: warp 4 + q holds TMEM lanes 32 q .. + 31
    const int q = warp & 3;
    const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16);
    const uint32_t lead_acce = PAIR ? peer_addr(acce, 0) : acce;
    float* part = reinterpret_cast<float*>(base);
    int cg = 0;
    bool ok = true;
    for (int tile = first; ok && tile < prm.tiles; tile += stride) {
      const int64_t row0 = tile_row(tile) + 32 * q, t0 = (int64_t)(tile / prm.mtiles) * NT;
      auto emit = [&](const float(&v)[16], int c) {   // columns c .. c + 15 of the tile
        if (split > 1) {   // the loads and MMAs of this CTA's only tile are complete: the rings are free
#pragma unroll
          for (int e = 0; e < 16; e++) part[(c + e) * 128 + 32 * q + lane] = v[e];
        } else {
          store_tile<16>(v, prm.alpha, prm.y, prm.dtype, row0, prm.out, t0 + c, prm.T);
        }
      };
      if constexpr (CHUNK) {
        float m[NT / 16][16];
#pragma unroll
        for (int c = 0; c < NT / 16; c++)
#pragma unroll
          for (int e = 0; e < 16; e++) m[c][e] = 0.0f;
        for (int g0 = s_begin; g0 < s_end; g0 += kChunkSteps, cg++) {
          const int b = cg & 1;
          if (!mbar_wait_warp(accf + 8 * b, (cg >> 1) & 1, abort, prm.waits.ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < NT / 16; c++) {
            float v[16];
            tmem_ld_cols(trow + b * NT + 16 * c, v);
#pragma unroll
            for (int e = 0; e < 16; e++) m[c][e] += v[e];
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (leader) mbar_arrive(acce + 8 * b);
            else mbar_arrive_remote(lead_acce + 8 * b);
          }
        }
        if (ok) {
#pragma unroll
          for (int c = 0; c < NT / 16; c++) emit(m[c], 16 * c);
        }
      } else {
        const int b = cg & 1;
        if (!mbar_wait_warp(accf + 8 * b, (cg >> 1) & 1, abort, prm.waits.ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < NT; c += 16) {
          float v[16];
          tmem_ld_cols(trow + b * NT + c, v);
          if (c + 16 == NT) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (leader) mbar_arrive(acce + 8 * b);
              else mbar_arrive_remote(lead_acce + 8 * b);
            }
          }
          emit(v, c);
        }
        cg++;
      }
    }
    if (!ok) fail();
  }
  __syncwarp();
  __syncthreads();
  if (PAIR) {
    cluster_sync();   // neither CTA touches the other's memory from here on
  } else if (split > 1) {
    cluster_sync();
    const int64_t t0 = (int64_t)(first / prm.mtiles) * NT;
    join_partials(base, rank, split, (int)min((int64_t)NT, prm.T - t0), tile_row(first), t0, prm.out, prm.alpha, prm.dtype,
                  prm.y);
    cluster_sync();
  }
  if (warp == 3) {
    tc_fence_after();
    tmem_free<PAIR>(tmem, C::kTmem);
  }
}

// x [T, K] -> bf16 parts [parts][T][Kp] that sum to x exactly.
template <typename S>
__global__ void __launch_bounds__(256) parts_kernel(const S* __restrict__ x, int64_t T, int64_t K, int64_t ld, int64_t Kp,
                                                    int parts, __nv_bfloat16* __restrict__ out) {
  const int64_t per = Kp / 8, total = T * per;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / per, k = (i - t * per) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = k + e < K ? float(x[t * ld + k + e]) : 0.0f;
    uint32_t w[3][4];
    cut_bf16<3>(v, w);
#pragma unroll
    for (int p = 0; p < 3; p++)
      if (p < parts) *reinterpret_cast<uint4*>(out + (p * T + t) * Kp + k) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
  }
}

int parts_of(int dtype) { return dtype == kMxBF16 ? 1 : dtype == kMxF16 ? 2 : 3; }

struct XView {
  const void* p;   // bf16
  int64_t rows, K, ld;
};

template <int FMT, int NT, bool PAIR, bool TR, bool CHUNK>
int launch_tiles(const XView& x, int parts, int64_t T, const Mx4View& w, float alpha, int dtype, void* y, int split,
                 cudaStream_t stream) {
  using C = Cfg<FMT, NT, PAIR, TR, CHUNK>;
  const int64_t pitch = mx4_pitch(w.n), groups = pitch / (FMT == kMXFP4 ? 64 : 32), wt = (w.rows + 127) / 128;
  CUtensorMap mw, ms, mx;
  if (!codes_map(&mw, w.codes, pitch, w.rows, 64, 128) || !scales_map(&ms, w.scales, wt * groups, C::kAtoms) ||
      !bf16_map(&mx, x.p, x.rows, x.K, x.ld, C::kXRows))
    return 5;
  LinParams p;
  p.y = y;
  p.T = T;
  p.out = TR ? w.n : w.rows;
  p.wrows = w.rows;
  p.alpha = alpha;
  p.dtype = dtype;
  p.parts = parts;
  p.nst = std::min(C::kMaxStages, C::kRing / (C::kA + parts * C::kB));
  p.turns = std::min(C::kGroups, p.nst);   // float16 in a pair: two stages
  p.ncs = C::kCS / C::kGroups * p.turns;
  p.steps = (int)((x.K + 127) / 128);
  p.groups = (int)groups;
  const int64_t mt = (p.out + 127) / 128;
  p.mtiles = (int)(PAIR ? (mt + 1) / 2 : mt);
  p.tiles = p.mtiles * (int)((T + NT - 1) / NT);
  p.waits = mx4_take_waits();
  const int sms = device_sm_count();
  const int grid = PAIR ? 2 * std::min(p.tiles, sms / 2) : split > 1 ? p.tiles * split : std::min(p.tiles, sms);
  return launch_cluster<mx4_linear_kernel<FMT, NT, PAIR, TR, CHUNK>>(grid, C::kThreads, C::kSmem, PAIR ? 2 : split, stream, mw,
                                                                    ms, mx, p, split);
}

template <int FMT, bool TR>
int launch_form(const XView& x, int parts, int64_t T, const Mx4View& w, float alpha, int dtype, void* y,
                cudaStream_t stream) {
  const int sms = device_sm_count();
  const int64_t mt = ((TR ? w.n : w.rows) + 127) / 128;
  const int steps = (int)((x.K + 127) / 128);
  // Clocks of a 128-deep step, from 4096 and 8192 columns with one round of tiles and cold weights: bf16 1320 to 1460
  // for any of the widths, which is the decoding's time, and 1750 in a pair.  (Float16's two parts take 1370, 1600
  // and 1880 for 32, 64 and 128 tokens and 3300 in a pair, float32's three with 64 tokens 2100; with these in the
  // estimates no case of 30 was faster and 300 tokens 4096 -> 14336 took 108 us for 99, so one pair of numbers
  // serves all.)
  if (dtype == kMxF32) {
    double clocks;
    const int split = best_split(mt * ((T + 63) / 64), steps, 1350, 64, sms, &clocks);
    return launch_tiles<FMT, 64, false, TR, true>(x, parts, T, w, alpha, dtype, y, split, stream);
  }
  int nt = 0, split = 1;
  double best = 0;
  for (int n = 32; n <= 128; n *= 2) {
    double clocks;
    const int s = best_split(mt * ((T + n - 1) / n), steps, 1350, n, sms, &clocks);
    if (nt == 0 || clocks < best) nt = n, split = s, best = clocks;
    if (n >= T) break;
  }
  const int64_t pairs = (mt + 1) / 2 * ((T + 255) / 256);
  if (T > 128 && (double)((pairs + sms / 2 - 1) / (sms / 2)) * steps * 1750 + 3500 <= best)
    return launch_tiles<FMT, 256, true, TR, false>(x, parts, T, w, alpha, dtype, y, 1, stream);
  switch (nt) {
    case 32: return launch_tiles<FMT, 32, false, TR, false>(x, parts, T, w, alpha, dtype, y, split, stream);
    case 64: return launch_tiles<FMT, 64, false, TR, false>(x, parts, T, w, alpha, dtype, y, split, stream);
    default: return launch_tiles<FMT, 128, false, TR, false>(x, parts, T, w, alpha, dtype, y, split, stream);
  }
}

// Whether the weights are decoded to the workspace first: for many tokens, where the decoded weights stay in
// L2 (126 MB) beside x and y, and for float32, whose sums in registers leave the fused form one group that
// decodes and 64 tokens a tile.  Measured, decoded first / in the product, us, cold weights:
//                             512 tokens   600          1024         4096
// 4096 -> 4096 (32 MiB)       33 / 29      34 / 37      34 / 38      99 / 124     MXFP4, bf16
//                             33 / 29      33 / 37      34 / 37      105 / 127    NVFP4, bf16
//                             33 / 29                   34 / 38      102 / 131    MXFP4, bf16, gradient
//                             56 / 39      58 / 59      62 / 62      222 / 233    MXFP4, f16
//                             56 / 39      57 / 59      62 / 62      228 / 238    NVFP4, f16
//                             57 / 39                   61 / 62      227 / 238    NVFP4, f16, gradient
// 4096 -> 14336 (112 MiB)                               129 / 120    433 / 425    MXFP4, bf16
//                                                       137 / 116    458 / 432    NVFP4, bf16
//                                                       227 / 206    748 / 718    MXFP4, f16
// float32 4096 -> 4096, 512 tokens 76 / 78; 4096 -> 14336, 1024 tokens 321 / 484.
bool use_dense(int dtype, int64_t T, int64_t rows, int64_t n) {
  return T > 544 && (dtype == kMxF32 || rows * n * 2 <= (int64_t)48 << 20);
}

// The device address of this unit's status word (looked up once per device).
int* status_word() {
  static std::atomic<int*> at[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  int* p = at[dev].load();
  if (!p && cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_status) == cudaSuccess) at[dev].store(p);
  return p;
}

int launch_dense(const XView& x, int parts, int64_t T, const Mx4View& w, float alpha, int dtype, int transpose, void* y,
                 void* wbuf, cudaStream_t stream) {
  const int64_t ld = (w.n + 7) / 8 * 8;
  if (int rc = launch_mx4_dequantize(w, 1.0f, kMxBF16, wbuf, ld, stream)) return rc;
  CUtensorMap mw, mx;
  if (!bf16_map(&mw, wbuf, w.rows, w.n, ld, transpose ? 64 : 128) || !bf16_map(&mx, x.p, x.rows, x.K, x.ld, 128)) return 5;
  dense::Params p;
  p.y = y;
  p.status = status_word();
  if (!p.status) return 6;
  p.T = T;
  p.out = transpose ? w.n : w.rows;
  p.alpha = alpha;
  p.dtype = dtype;
  p.parts = parts;
  p.nst = dense::kRing / ((1 + parts) * dense::kBox);
  p.steps = (int)((x.K + 63) / 64);
  p.chunk = dtype == kMxF32 ? 1 : p.steps;
  p.mtiles = (int)((p.out + 255) / 256);
  p.tiles = p.mtiles * (int)((T + 255) / 256);
  p.waits = mx4_take_waits();
  const int grid = 2 * std::min(p.tiles, device_sm_count() / 2);
  return transpose ? launch_cluster<dense::dense_kernel<true>>(grid, dense::kThreads, dense::kSmem, 2, stream, mw, mx, p)
                   : launch_cluster<dense::dense_kernel<false>>(grid, dense::kThreads, dense::kSmem, 2, stream, mw, mx, p);
}

int64_t parts_pitch(int64_t K) { return (K + 7) / 8 * 8; }

}  // namespace

namespace {
size_t parts_bytes(int dtype, int64_t T, int64_t K, int aligned) {
  return dtype == kMxBF16 && aligned ? 0 : ((size_t)parts_of(dtype) * T * parts_pitch(K) * 2 + 255) / 256 * 256;
}
}  // namespace

size_t mx4_linear_workspace_bytes(int dtype, int64_t T, int64_t rows, int64_t n, int aligned, int transpose) {
  if (!transpose && mx4_stream_applies(dtype, T, rows, n)) return mx4_stream_workspace_bytes(dtype, T, rows, n);
  return parts_bytes(dtype, T, transpose ? rows : n, aligned) +
         (use_dense(dtype, T, rows, n) ? (size_t)rows * ((n + 7) / 8 * 8) * 2 : 0);
}

int launch_mx4_linear(int dtype, const void* x, int64_t T, int64_t ld, int aligned, const Mx4View& w, float alpha,
                      int transpose, void* y, void* ws, cudaStream_t stream) {
  if (!bind_context()) return 6;
  if (!transpose && mx4_stream_applies(dtype, T, w.rows, w.n))
    return launch_mx4_stream(dtype, x, T, ld, aligned, w, alpha, y, ws, stream);
  const int64_t K = transpose ? w.rows : w.n;
  const int parts = parts_of(dtype);
  XView xv{x, T, K, T == 1 ? parts_pitch(K) : ld};   // one row has no pitch of its own
  const size_t pb = parts_bytes(dtype, T, K, aligned);
  if (pb > 0) {
    const int64_t Kp = parts_pitch(K);
    const unsigned grid = (unsigned)std::min<int64_t>((T * (Kp / 8) + 255) / 256, (int64_t)device_sm_count() * 8);
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(ws);
    if (dtype == kMxBF16) parts_kernel<<<grid, 256, 0, stream>>>(static_cast<const __nv_bfloat16*>(x), T, K, ld, Kp, parts, out);
    else if (dtype == kMxF16) parts_kernel<<<grid, 256, 0, stream>>>(static_cast<const __half*>(x), T, K, ld, Kp, parts, out);
    else parts_kernel<<<grid, 256, 0, stream>>>(static_cast<const float*>(x), T, K, ld, Kp, parts, out);
    note_launch();
    xv = XView{ws, parts * T, K, Kp};
  }
  if (use_dense(dtype, T, w.rows, w.n))
    return launch_dense(xv, parts, T, w, alpha, dtype, transpose, y, static_cast<uint8_t*>(ws) + pb, stream);
  if (w.fmt == kMXFP4)
    return transpose ? launch_form<kMXFP4, true>(xv, parts, T, w, alpha, dtype, y, stream)
                     : launch_form<kMXFP4, false>(xv, parts, T, w, alpha, dtype, y, stream);
  return transpose ? launch_form<kNVFP4, true>(xv, parts, T, w, alpha, dtype, y, stream)
                   : launch_form<kNVFP4, false>(xv, parts, T, w, alpha, dtype, y, stream);
}

int mx4_linear_status(cudaStream_t stream, int* status) { return read_status_word(g_status, stream, status); }

}  // namespace cpk
