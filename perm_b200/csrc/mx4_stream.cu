// y = alpha * x w^T for a few tokens: the weights stream once from HBM, 17/32 or 9/16 of a byte each,
// and everything else has to keep up with that.
//
// At 6.5 TB/s an SM gets about 44 weights a clock and issues 128 lane instructions, so a weight has
// less than three.  Decoding to bf16 (five instructions for two weights) and storing the tile for
// tcgen05 does not fit; here the weights go straight into registers as f16, one conversion for
// two, and through mma.sync m16n8k16 with 16 rows of weights as the A operand and up to 8 tokens as B (more
// tokens: more B tiles).  ldmatrix hands lane (g, t) the word of eight codes 8t .. 8t + 7 of a 32-code
// block of row g; which k of the MMA a code sits on is free as long as x is taken in the same order, and
// with that order the eight values of x that a lane needs are 16 neighbouring bytes.
//
//   MXFP4  The two MMAs of a block start from zero; their sums are multiplied by the block's power of two
//          and added in float32, exact for every scale.
//   NVFP4  A lane's codes lie in one block of 16; code times scale has six significant bits and fits f16,
//          so the A registers are multiplied before the MMA, which then accumulates 256 columns.
//
// Activations are f16 too.  float16 is taken as it is.  bf16 and float32 rows are multiplied by a power of
// two that brings the row's largest magnitude (of this CTA's columns) to [2^14, 2^15): a bf16 value is then
// exact unless it is below 2^-32 of the largest, and off by at most 2^-40 of the largest otherwise.
// float32 values are the sum of two f16 parts, the second 2^11 times finer, to within 2^-23 of each value.
//
// Every row tile needs x converted.  Where that is a large part of the work a first kernel converts it once,
// into the workspace; the product is launched so that it may start beside that kernel (programmatic
// dependent launch), brings its first weights in and waits for it only before it reads x.
//
// A CTA holds 128 rows (16 for each of eight warps) and a slice of the columns; a cluster of up to eight
// shares a row tile and joins the partial sums through distributed shared memory in rank order.  Codes
// and scale tiles arrive by TMA in stages of 256 columns; x is converted into shared memory while the first
// stages are in flight.  Two CTAs fit an SM.
#include <type_traits>
#include "mx4_product.cuh"

namespace cpk {
namespace {

__device__ int g_status;

constexpr unsigned long long kWaitNs = 1000000000ull;
constexpr int kWarps = 8;
constexpr int kThreads = 32 * (kWarps + 1);   // the last warp loads
constexpr int kMaxStages = 6;

struct StreamParams {
  const void* x;
  void* y;
  int64_t T, K, ld, rows;
  float alpha;
  int dtype;
  int steps, nst;       // 256-column steps; stages of the ring
  int slice;            // columns of the widest slice (the pitch of the converted x)
  int groups;           // scale tiles per 128 rows
  int vec;              // x's rows start on 16-byte boundaries
  const uint32_t* top;  // converted x: the rows' largest magnitudes
  int64_t pitch;        // and its bytes per row
};

__device__ __forceinline__ void ldmatrix4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
// Eight codes -> four f16 pairs.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t (&v)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
      : "r"(w));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Two e8m0 scales (low half of w) -> float32.
__device__ __forceinline__ void e8m0x2(uint32_t w, float& lo, float& hi) {
  uint32_t r;
  asm("{\n\t.reg .b16 s;\n\tcvt.u16.u32 s, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, s;\n\t}" : "=r"(r) : "r"(w));
  lo = __uint_as_float(r << 16);
  hi = __uint_as_float(r & 0xFFFF0000u);
}
// Two e4m3 scales (low half of w, signs cleared) -> f16.
__device__ __forceinline__ uint32_t e4m3x2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 s;\n\tcvt.u16.u32 s, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, s;\n\t}" : "=r"(r) : "r"(w));
  return r;
}

__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_f32(__half v) { return __half2float(v); }

template <typename S> struct Parts { static constexpr int k = 1; static constexpr bool scaled = true; };
template <> struct Parts<__half> { static constexpr int k = 1; static constexpr bool scaled = false; };
template <> struct Parts<float> { static constexpr int k = 2; static constexpr bool scaled = true; };

// Unit c of a row t, `units` to a row.
struct Unit {
  int t, c;
  __device__ __forceinline__ Unit(int i, int units) : t(0), c(i) { wrap(units); }
  __device__ __forceinline__ void next(int by, int units) {
    c += by;
    wrap(units);
  }
  __device__ __forceinline__ void wrap(int units) {
    while (c >= units) c -= units, t++;
  }
};
// Eight values of x in shared memory.
template <typename S> __device__ __forceinline__ void read_x8(const uint8_t* at, float (&v)[8]) {
  constexpr int W = sizeof(S) / 2;
  uint4 w[W];
#pragma unroll
  for (int i = 0; i < W; i++) w[i] = reinterpret_cast<const uint4*>(at)[i];
  const S* e = reinterpret_cast<const S*>(w);
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = as_f32(e[i]);
}
// The largest finite magnitude of eight values, as float32 bits.
template <typename S> __device__ __forceinline__ uint32_t top_x8(const uint8_t* at) {
  if (sizeof(S) == 2) {   // bf16: two at a time; a NaN or infinity shows in the maximum and takes the long way
    const uint4 w = *reinterpret_cast<const uint4*>(at);
    const uint32_t two = __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
    const uint32_t m = max(two >> 16, two & 0xFFFFu);
    if (m < 0x7F80u) return m << 16;
  }
  float v[8];
  read_x8<S>(at, v);
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const uint32_t b = __float_as_uint(v[e]) & 0x7FFFFFFFu;
    m = max(m, b < 0x7F800000u ? b : 0u);
  }
  return m;
}

// 2^(14 - e) for a largest magnitude (as bits) of exponent e, and its inverse.
__device__ __forceinline__ float scale_up(uint32_t top) {
  return __uint_as_float((uint32_t)min(268 - max((int)(top >> 23), 1), 247) << 23);
}
__device__ __forceinline__ float scale_down(uint32_t top) {
  return __uint_as_float((uint32_t)max(max((int)(top >> 23), 1) - 14, 7) << 23);
}
// Eight values, scaled, as f16 parts at `at` (16 bytes each).
template <typename S> __device__ __forceinline__ void write_x8(uint8_t* at, const float (&v)[8], float up) {
  constexpr int P = Parts<S>::k;
  uint32_t w[P][4];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float a = v[e] * up, b = v[e + 1] * up;
    const __half2 h = __floats2half2_rn(a, b);
    w[0][e / 2] = *reinterpret_cast<const uint32_t*>(&h);
    if (P == 2) {   // of an infinity or NaN the first part holds it all
      const float2 f = __half22float2(h);
      const float ra = fabsf(a) < 1e30f ? (a - f.x) * 2048.0f : 0.0f, rb = fabsf(b) < 1e30f ? (b - f.y) * 2048.0f : 0.0f;
      const __half2 l = __floats2half2_rn(ra, rb);
      w[P - 1][e / 2] = *reinterpret_cast<const uint32_t*>(&l);
    }
  }
#pragma unroll
  for (int p = 0; p < P; p++) reinterpret_cast<uint4*>(at)[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}

// One CTA per row of x: the row's largest magnitude, and the row as scaled f16 parts, [eight
// columns][part], zero from K to the padded end.
template <typename S>
__global__ void __launch_bounds__(512) convert_kernel(const S* __restrict__ x, int64_t K, int64_t ld, int vec, int groups,
                                                      uint8_t* __restrict__ out, uint32_t* __restrict__ top) {
  __shared__ uint32_t most;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = blockIdx.x;
  const S* row = x + t * ld;
  auto load = [&](int c, float (&v)[8]) {
    const int64_t left = K - (int64_t)c * 8;
    if (vec && left >= 8) {
      read_x8<S>(reinterpret_cast<const uint8_t*>(row + c * 8), v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = e < left ? as_f32(row[c * 8 + e]) : 0.0f;
    }
  };
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  uint32_t m = 0;
#pragma unroll 4
  for (int c = threadIdx.x; c < groups; c += 512) {
    float v[8];
    load(c, v);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t b = __float_as_uint(v[e]) & 0x7FFFFFFFu;
      m = max(m, b < 0x7F800000u ? b : 0u);
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (threadIdx.x % 32 == 0) atomicMax(&most, m);
  __syncthreads();
  if (threadIdx.x == 0) top[t] = most;
  const float up = scale_up(most);
#pragma unroll 4
  for (int c = threadIdx.x; c < groups; c += 512) {
    float v[8];
    load(c, v);
    write_x8<S>(out + ((int64_t)t * groups + c) * (16 * Parts<S>::k), v, up);
  }
}

// DONE: x is what convert_kernel left.
template <int FMT, int NB, typename S, bool DONE>
__global__ void __launch_bounds__(kThreads, 2)
    mx4_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_s,
                      const StreamParams prm, int split) {
  constexpr int NTOK = 8 * NB, P = Parts<S>::k;
  constexpr bool kScaled = Parts<S>::scaled;
  constexpr int kAtoms = FMT == kMXFP4 ? 2 : 4;          // scale tiles of 128 rows x 256 columns
  constexpr int kStage = 128 * 128 + kAtoms * 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int nst = prm.nst;
  // bytes of a token's slice; the odd end keeps eight lanes' 16-byte reads (two tokens, four groups) on
  // different banks
  const int xpitch = prm.slice * 2 * P + (P == 1 ? 64 : 16);
  uint8_t* xs = base + nst * kStage;                     // [token][eight columns][part] f16
  uint32_t* top = reinterpret_cast<uint32_t*>(xs + prm.T * xpitch);   // largest magnitudes, as bits
  uint64_t* bars = reinterpret_cast<uint64_t*>(top + NTOK);
  volatile int* misc = reinterpret_cast<volatile int*>(bars + 2 * kMaxStages);   // [0] abort
  const uint32_t ring = smem_u32(base), full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int tile = (int)blockIdx.x / split;
  const int s_begin = (int)((int64_t)prm.steps * rank / split), s_end = (int)((int64_t)prm.steps * (rank + 1) / split);
  const int T = (int)prm.T;
  volatile int* abort = &misc[0];

  if (threadIdx.x == 0) {
    for (int s = 0; s < nst; s++) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, kWarps);
    }
    misc[0] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < NTOK) top[threadIdx.x] = 0;
  __syncthreads();

  float acc[NB][4];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[b][e] = 0.0f;

  if (warp == kWarps) {
    if (lane == 0) {
      Ring rg{0, 0};
      bool ok = true;
      int loads = 0;
      for (int s = s_begin; s < s_end; s++, loads++) {
        if (loads >= nst && !mbar_wait(empty0 + 8 * rg.st, rg.ph ^ 1, abort, kWaitNs)) {
          ok = false;
          break;
        }
        const uint32_t fb = full0 + 8 * rg.st, sw = ring + rg.st * kStage;
        mbar_expect_tx(fb, kStage);
        tma_load(sw, &map_w, s * 128, tile * 128, fb);
        tma_load(sw + 128 * 128, &map_s, 0, tile * prm.groups + s * kAtoms, fb);
        rg.advance(nst);
      }
      if (!ok) fail_cta(abort, &g_status);
      for (int k = min(loads, nst); k > 0; k--) {   // every load issued lands before the CTA goes on
        rg.back(nst);
        int zero = 0;
        mbar_wait(full0 + 8 * rg.st, rg.ph, &zero, kWaitNs);
      }
    }
  } else {
    // ---- x into shared memory: asynchronous copies of the rows as they are, then (scaled types) a pass
    // for the largest magnitudes and one that converts each group of eight values in place.  A warp takes
    // units of 256 columns of one row; a thread reads back only what it copied itself.
    const int units = s_end - s_begin;   // a row's
    const int64_t k0 = (int64_t)s_begin * 256;
    Unit u(warp, units);
    if (DONE) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      if (threadIdx.x < T) top[threadIdx.x] = __ldcg(prm.top + threadIdx.x);
      for (; u.t < T; u.next(kWarps, units)) {
        const int c = u.c * 32 + lane;
        const uint8_t* src = static_cast<const uint8_t*>(prm.x) + u.t * prm.pitch + (k0 / 8 + c) * (16 * P);
#pragma unroll
        for (int p = 0; p < P; p++)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(xs) + u.t * xpitch + (c * P + p) * 16),
                       "l"(src + 16 * p)
                       : "memory");
      }
    } else {
      for (; u.t < T; u.next(kWarps, units)) {
        const int c = u.c * 32 + lane;   // group of eight columns
        const int64_t left = prm.K - k0 - (int64_t)c * 8;   // values of the row from here on
        const S* src = static_cast<const S*>(prm.x) + u.t * prm.ld + k0 + c * 8;
        uint8_t* dst = xs + u.t * xpitch + c * (16 * P);
        if (prm.vec) {   // 16 bytes at a time: sources past the row's end stay at x, which is aligned as its rows are
#pragma unroll
          for (int p = 0; p < P; p++) {
            const int64_t bytes = (left - p * (8 / P)) * (int64_t)sizeof(S);
            const uint32_t n = bytes >= 16 ? 16 : bytes > 0 ? (uint32_t)bytes : 0;   // the rest is zero
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst) + 16 * p),
                         "l"(n ? src + p * (8 / P) : static_cast<const S*>(prm.x)), "r"(n)
                         : "memory");
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) reinterpret_cast<S*>(dst)[e] = e < left ? src[e] : S(0.0f);
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (kScaled && !DONE) {
      for (u = Unit(warp, units); u.t < T; u.next(kWarps, units)) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, top_x8<S>(xs + u.t * xpitch + (u.c * 32 + lane) * (16 * P)));
        if (lane == 0) atomicMax(&top[u.t], m);
      }
      asm volatile("bar.sync 1, %0;" ::"r"(32 * kWarps) : "memory");
      for (u = Unit(warp, units); u.t < T; u.next(kWarps, units)) {
        uint8_t* at = xs + u.t * xpitch + (u.c * 32 + lane) * (16 * P);
        float v[8];
        read_x8<S>(at, v);
        write_x8<S>(at, v, scale_up(top[u.t]));
      }
    }
    asm volatile("bar.sync 1, %0;" ::"r"(32 * kWarps) : "memory");

    // ---- the weights
    const int g = lane >> 2, t4 = lane & 3;
    float down[NB][2];   // undoes `up` for this lane's two tokens of each tile
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int e = 0; e < 2; e++)
        down[b][e] = kScaled ? scale_down(top[8 * b + 2 * t4 + e]) : 1.0f;
    const uint32_t row_at = (16 * warp + (lane & 7)) * 128, x7 = lane & 7;
    const uint32_t srow = ((16 * warp + g) & 31) * 16 + ((16 * warp + g) >> 5) * 4;   // row g's scale word; row g + 8: + 128
    // tokens past the last read a row that is there; their results are not used
    uint32_t xlane[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) xlane[b] = smem_u32(xs) + (8 * b + g < T ? 8 * b + g : 0) * xpitch + t4 * (16 * P);
    Ring rg{0, 0};
    bool ok = true;
    for (int s = s_begin; s < s_end; s++) {
      if (!mbar_wait_warp(full0 + 8 * rg.st, rg.ph, abort, kWaitNs)) {
        ok = false;
        break;
      }
      const uint32_t sw = ring + rg.st * kStage;
      const uint32_t sc = sw + 128 * 128;
      const uint32_t xcol = (s - s_begin) * (512 * P);
      float c[P][NB][4];
      if (FMT == kNVFP4) {
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
          for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) c[p][b][e] = 0.0f;
      }
#pragma unroll
      for (int half = 0; half < 2; half++) {   // 128 columns
        uint32_t wa[4], wb[4];
        const uint32_t at = sw + row_at + (((half * 4 + (lane >> 3)) ^ x7) << 4);
        ldmatrix4(at, wa);               // rows g: words of four blocks of 32
        ldmatrix4(at + 8 * 128, wb);     // rows g + 8
        float sa[4], sb[4];
        uint32_t ha[4], hb[4];
        if (FMT == kMXFP4) {
          const uint32_t va = ld_stage_u32(sc + half * 512 + srow);
          const uint32_t vb = ld_stage_u32(sc + half * 512 + srow + 128);
          e8m0x2(va, sa[0], sa[1]);
          e8m0x2(va >> 16, sa[2], sa[3]);
          e8m0x2(vb, sb[0], sb[1]);
          e8m0x2(vb >> 16, sb[2], sb[3]);
        } else {
          const uint32_t sel = t4 < 2 ? 0x1010u : 0x3232u;   // this lane's block of a pair
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const uint32_t va = ld_stage_u32(sc + (half * 2 + j / 2) * 512 + srow) & 0x7F7F7F7Fu;
            const uint32_t vb = ld_stage_u32(sc + (half * 2 + j / 2) * 512 + srow + 128) & 0x7F7F7F7Fu;
            ha[j] = __byte_perm(e4m3x2(va), 0, sel);
            ha[j + 1] = __byte_perm(e4m3x2(va >> 16), 0, sel);
            hb[j] = __byte_perm(e4m3x2(vb), 0, sel);
            hb[j + 1] = __byte_perm(e4m3x2(vb >> 16), 0, sel);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          uint32_t a[4], b[4];
          codes_f16(wa[j], a);
          codes_f16(wb[j], b);
          if (FMT == kNVFP4) {
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = mul_f16x2(a[i], ha[j]), b[i] = mul_f16x2(b[i], hb[j]);
          }
#pragma unroll
          for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int p = 0; p < P; p++) {
              uint4 xv;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(xv.x), "=r"(xv.y), "=r"(xv.z), "=r"(xv.w)
                           : "r"(xlane[nb] + xcol + (half * 256 + j * 64) * P + p * 16));
              float(&d)[4] = c[p][nb];
              if (FMT == kMXFP4) mma_f16_zero(d, a[0], b[0], a[1], b[1], xv.x, xv.y);
              else mma_f16(d, a[0], b[0], a[1], b[1], xv.x, xv.y);
              mma_f16(d, a[2], b[2], a[3], b[3], xv.z, xv.w);
              if (FMT == kMXFP4) {
                const float fine = p == 1 ? 1.0f / 2048.0f : 1.0f;
                const float d0 = kScaled ? d[0] * (down[nb][0] * fine) : d[0], d1 = kScaled ? d[1] * (down[nb][1] * fine) : d[1];
                const float d2 = kScaled ? d[2] * (down[nb][0] * fine) : d[2], d3 = kScaled ? d[3] * (down[nb][1] * fine) : d[3];
                acc[nb][0] += d0 * sa[j];
                acc[nb][1] += d1 * sa[j];
                acc[nb][2] += d2 * sb[j];
                acc[nb][3] += d3 * sb[j];
              }
            }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty0 + 8 * rg.st);
      rg.advance(nst);
      if (FMT == kNVFP4) {
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int p = 0; p < P; p++) {
            const float fine = p == 1 ? 1.0f / 2048.0f : 1.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) acc[nb][e] += c[p][nb][e] * (down[nb][e & 1] * fine);
          }
      }
    }
    if (!ok) fail_cta(abort, &g_status);
  }
  // ---- results: lane (g, t) has rows g, g + 8 of its warp's 16 and tokens 2t, 2t + 1 of each tile
  const int64_t row0 = (int64_t)tile * 128;
  if (split > 1) {
    __syncthreads();   // all loads have landed and been read: the ring is free
    float* part = reinterpret_cast<float*>(base);
    if (warp < kWarps) {
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          part[(8 * nb + 2 * (lane & 3) + (e & 1)) * 128 + 16 * warp + (lane >> 2) + (e >> 1) * 8] = acc[nb][e];
    }
    cluster_sync();
    join_partials(base, rank, split, T, row0, 0, prm.rows, prm.alpha, prm.dtype, prm.y);
    cluster_sync();
  } else if (warp < kWarps) {
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int t = 8 * nb + 2 * (lane & 3) + (e & 1);
        const int64_t row = row0 + 16 * warp + (lane >> 2) + (e >> 1) * 8;
        if (t < T && row < prm.rows) put_out(prm.y, prm.dtype, t * prm.rows + row, prm.alpha * acc[nb][e]);
      }
  }
}

template <int FMT, int NB, typename S, bool DONE>
int launch_tiles(StreamParams& p, const Mx4View& w, int split, cudaStream_t stream) {
  constexpr int kAtoms = FMT == kMXFP4 ? 2 : 4, kStage = 128 * 128 + kAtoms * 512;
  const int64_t pitch = mx4_pitch(w.n), wt = (w.rows + 127) / 128;
  CUtensorMap mw, ms;
  if (!codes_map(&mw, w.codes, pitch, w.rows, 128, 128) || !scales_map(&ms, w.scales, wt * p.groups, kAtoms)) return 5;
  const size_t smem = 1024 + (size_t)p.nst * kStage + (size_t)p.T * (p.slice * 2 * Parts<S>::k + 64) + 8 * NB * 4 +
                      16 * kMaxStages + 64;
  return launch_cluster_after<mx4_stream_kernel<FMT, NB, S, DONE>>(DONE, (int)wt * split, kThreads, smem, split, stream, mw,
                                                                  ms, p, split);
}

struct StreamPlan {
  int split, nst, slice;
  bool convert;         // x is converted by a kernel of its own
};
// False where the kernel does not take these sizes: more tokens than it is good for (MXFP4, bf16, here / decoded
// to bf16 for tcgen05: 4096 -> 14336 with 16 tokens 18 / 23 us, with 24 tokens 33 / 23 us), or slices of x
// that would leave no room in shared memory.
bool stream_plan(int dtype, int64_t T, int64_t rows, int64_t n, StreamPlan* plan) {
  if (T > 16) return false;
  const int64_t wt = (rows + 127) / 128;
  // The converting kernel costs a launch.  4096 -> 14336, bf16, with it / without: 4 tokens 12.0 / 12.3 us, 8
  // tokens 12.7 / 14.7, 16 tokens 18 / 24; 4096 -> 4096 with 8 tokens 7.2 / 7.0.
  const bool convert = dtype != kMxF16 && T * n * wt > 2000000;
  const int parts = dtype == kMxF32 ? 2 : 1;
  const int most = 2;   // CTAs to an SM, by registers (three of fewer registers were 3 % slower for one token)
  const int sms = device_sm_count();
  const int steps = (int)(mx4_pitch(n) / 128), stage = 128 * 128 + 4 * 512;   // NVFP4's; MXFP4's is smaller
  int split = 1;
  // one and a half rounds of shorter CTAs beat one of longer ones (14336 -> 4096, one token: 9.7 / 10.9 us)
  while (split < 8 && wt <= 3 * most / 2 * cluster_slots(split * 2, sms) && split * 2 <= steps) split *= 2;
  // x's slice stays in shared memory beside at least two stages
  auto x_bytes = [&](int sp) { return T * ((int64_t)(steps + sp - 1) / sp * 512 * parts + 64); };
  const int64_t room = 222 * 1024;
  while (split < 8 && split * 2 <= steps && x_bytes(split) + 2 * stage > room / most) split *= 2;
  if (x_bytes(split) + 2 * stage > (T <= 8 ? room : room / 2)) return false;
  // as many CTAs to an SM as leaves each two stages
  const int mine = (steps + split - 1) / split;
  int nst = 0;
  for (int ctas = most; ctas > 0 && nst < std::min(2, mine); ctas--)
    nst = (int)((room / ctas - 2048 - x_bytes(split)) / stage);
  *plan = StreamPlan{split, std::min(std::min(nst, kMaxStages), mine), mine * 256, convert};
  return true;
}

template <int FMT, typename S, bool DONE>
int launch_tokens(StreamParams& p, const Mx4View& w, int split, cudaStream_t stream) {
  if (p.T <= 8) return launch_tiles<FMT, 1, S, DONE>(p, w, split, stream);
  return launch_tiles<FMT, 2, S, DONE>(p, w, split, stream);
}

template <int FMT, typename S>
int launch_type(StreamParams& p, const Mx4View& w, int split, bool convert, void* ws, cudaStream_t stream) {
  if constexpr (Parts<S>::scaled) {
    if (convert) {
      const int groups = p.steps * 32;
      p.pitch = (int64_t)groups * 16 * Parts<S>::k;
      uint8_t* out = static_cast<uint8_t*>(ws);
      uint32_t* top = reinterpret_cast<uint32_t*>(out + p.T * p.pitch);
      convert_kernel<S><<<(unsigned)p.T, 512, 0, stream>>>(static_cast<const S*>(p.x), p.K, p.ld, p.vec, groups, out, top);
      note_launch();
      p.x = out;
      p.top = top;
      return launch_tokens<FMT, S, true>(p, w, split, stream);
    }
  }
  return launch_tokens<FMT, S, false>(p, w, split, stream);
}

}  // namespace

bool mx4_stream_applies(int dtype, int64_t T, int64_t rows, int64_t n) {
  StreamPlan plan;
  return stream_plan(dtype, T, rows, n, &plan);
}

size_t mx4_stream_workspace_bytes(int dtype, int64_t T, int64_t rows, int64_t n) {
  StreamPlan plan;
  if (!stream_plan(dtype, T, rows, n, &plan) || !plan.convert) return 0;
  return (size_t)T * (mx4_pitch(n) / 128 * 32 * 16 * (dtype == kMxF32 ? 2 : 1) + 4);
}

int launch_mx4_stream(int dtype, const void* x, int64_t T, int64_t ld, int aligned, const Mx4View& w, float alpha, void* y,
                      void* ws, cudaStream_t stream) {
  StreamPlan plan;
  if (!stream_plan(dtype, T, w.rows, w.n, &plan)) return 6;
  const int steps = (int)(mx4_pitch(w.n) / 128);
  StreamParams p = {};
  p.x = x;
  p.y = y;
  p.T = T;
  p.K = w.n;
  p.ld = ld;
  p.rows = w.rows;
  p.alpha = alpha;
  p.dtype = dtype;
  p.steps = steps;
  p.nst = plan.nst;
  p.slice = plan.slice;
  p.groups = steps * (w.fmt == kMXFP4 ? 2 : 4);
  p.vec = aligned;
  if (w.fmt == kMXFP4) {
    if (dtype == kMxBF16) return launch_type<kMXFP4, __nv_bfloat16>(p, w, plan.split, plan.convert, ws, stream);
    if (dtype == kMxF16) return launch_type<kMXFP4, __half>(p, w, plan.split, plan.convert, ws, stream);
    return launch_type<kMXFP4, float>(p, w, plan.split, plan.convert, ws, stream);
  }
  if (dtype == kMxBF16) return launch_type<kNVFP4, __nv_bfloat16>(p, w, plan.split, plan.convert, ws, stream);
  if (dtype == kMxF16) return launch_type<kNVFP4, __half>(p, w, plan.split, plan.convert, ws, stream);
  return launch_type<kNVFP4, float>(p, w, plan.split, plan.convert, ws, stream);
}

int mx4_stream_status(cudaStream_t stream, int* status) { return read_status_word(g_status, stream, status); }

}  // namespace cpk
