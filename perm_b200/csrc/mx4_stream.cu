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
//   MXFP4  The two MMAs of a block start from zero; their sums are multiplied by the row's unit (below) and
//          the block's power of two and added in float32.
//   NVFP4  A lane's codes lie in one block of 16; code times scale has six significant bits and fits f16,
//          so the A registers are multiplied before the MMA, which then accumulates 256 columns.
//
// Activations are f16 too.  float16 is taken as it is.  bf16 and float32 rows are taken in a unit, the power
// of two that brings the row's largest magnitude to [2^14, 2^15).  A bf16 value is then exact if it is at least
// 2^-31 of the largest.  A float32 value is the sum of two f16 parts, the second 2^11 times finer: 23 bits
// and a sign, so that it is off by a unit in the last place (2^-23 of itself) at most if it is at least 2^-26 of the
// largest.  (A third part makes it exact, and 8 tokens 4096 -> 14336 28 us for 16.5.)  A part is a column of B of
// its own.  Units of 2^-126 to 2^49 keep every step inside float32's range unless the result is outside.
//
// Where a row has smaller values, or a larger unit, the CTA takes all its rows as they are instead, in bf16: weights
// times scales, exact as in the products for more tokens, against bf16 values or the three bf16 parts that a
// float32 is cut into, so that nothing is lost beside a large value.  Four more instructions for two weights, and
// the cutting, make that the slower way (one token 4096 -> 14336: bf16 14.0 us for 10.1, float32 27 for 12).
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
  const void* units;    // x as convert_kernel left it
  const uint32_t* top;  // its rows' largest magnitudes
  int64_t pitch;        // and its bytes per row
  Mx4Waits waits;
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
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A pair of f16 of at most eight significant bits -> bf16: the upper halves of their float32 values.
__device__ __forceinline__ uint32_t f16_to_bf16(uint32_t h) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x7632);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Two e8m0 scales (low half of w) -> bf16.
__device__ __forceinline__ uint32_t e8m0x2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 s;\n\tcvt.u16.u32 s, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, s;\n\t}" : "=r"(r) : "r"(w));
  return r;
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

// k: parts.  least: the exponent, in the row's unit, from which a value is held.
template <typename S> struct Parts { static constexpr int k = 1, least = -17; static constexpr bool scaled = true; };
template <> struct Parts<__half> { static constexpr int k = 1, least = 0; static constexpr bool scaled = false; };
template <> struct Parts<float> { static constexpr int k = 2, least = -12; static constexpr bool scaled = true; };

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
// Eight values of x, 16 bytes at a time, `apart` bytes from one another.
template <typename S> __device__ __forceinline__ void read_x8(const uint8_t* at, int apart, float (&v)[8]) {
  constexpr int W = sizeof(S) / 2;
  uint4 w[W];
#pragma unroll
  for (int i = 0; i < W; i++) w[i] = *reinterpret_cast<const uint4*>(at + i * apart);
  const S* e = reinterpret_cast<const S*>(w);
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = as_f32(e[i]);
}
// Of some values, as float32 bits: the largest finite magnitude (0: none), one less than the least magnitude that
// is not zero (all ones: none), and whether one is infinite or NaN.
struct Range {
  uint32_t top = 0, low = 0xFFFFFFFFu;
  bool odd = false;
  __device__ __forceinline__ void take(float v) {
    const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
    const bool is_odd = b >= 0x7F800000u;
    odd |= is_odd;
    top = max(top, is_odd ? 0u : b);
    low = min(low, b - 1);
  }
};
// With eight values of x in shared memory.
template <typename S> __device__ __forceinline__ void take_x8(const uint8_t* at, int apart, Range& r) {
  if (sizeof(S) == 2) {   // bf16: two at a time; a NaN or infinity shows in the maximum and takes the long way
    const uint4 w = *reinterpret_cast<const uint4*>(at);
    const uint32_t two = __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
    const uint32_t m = max(two >> 16, two & 0xFFFFu);
    if (m < 0x7F80u) {
      // one less than each half's magnitude: the upper bit, set meanwhile, keeps a borrow inside its half
      auto less = [](uint32_t v) { return ((v | 0x80008000u) - 0x00010001u) ^ 0x80008000u; };
      const uint32_t l2 = __vminu2(__vminu2(less(w.x), less(w.y)), __vminu2(less(w.z), less(w.w)));
      const uint32_t l = min(l2 >> 16, l2 & 0xFFFFu);
      r.top = max(r.top, m << 16);
      r.low = min(r.low, ((l + 1) << 16) - 1);   // l = 0xFFFF, no value but zeros: all ones
      return;
    }
  }
  float v[8];
  read_x8<S>(at, apart, v);
#pragma unroll
  for (int e = 0; e < 8; e++) r.take(v[e]);
}
// The exponent of one over a row's unit, for a largest magnitude (as bits) with the exponent field e: the largest
// goes to [2^14, 2^15), or as far as 2^126 takes it.
__device__ __forceinline__ int unit_shift(uint32_t top) { return min(141 - (int)(top >> 23), 126); }
// Whether a row's unit holds all its values.
template <typename S> __device__ __forceinline__ bool in_unit(uint32_t top, uint32_t low) {
  const int e = (int)(top >> 23), least = (int)((low + 1) >> 23);
  return top == 0 || (e <= 127 + 63 && least > 0 && least - 127 + unit_shift(top) >= Parts<S>::least);
}
// One over the unit of a row that its unit holds, and the unit.  1 for no magnitude.
__device__ __forceinline__ float scale_up(uint32_t top) {
  return top ? __uint_as_float((uint32_t)(127 + unit_shift(top)) << 23) : 1.0f;
}
__device__ __forceinline__ float scale_down(uint32_t top) {
  return top ? __uint_as_float((uint32_t)(127 - unit_shift(top)) << 23) : 1.0f;
}
// Eight values in their row's unit (`up`) as f16, the parts of a value `apart` bytes from one another.
template <typename S> __device__ __forceinline__ void write_x8(uint8_t* at, int64_t apart, const float (&v)[8], float up) {
  constexpr int P = Parts<S>::k;
  uint32_t w[P][4];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float a = v[e] * up, b = v[e + 1] * up;
#pragma unroll
    for (int p = 0; p < P; p++) {
      const __half2 h = __floats2half2_rn(a, b);
      w[p][e / 2] = *reinterpret_cast<const uint32_t*>(&h);
      const float2 f = __half22float2(h);   // what is left, 2^11 times finer; of an infinity or NaN the first part holds it all
      a = fabsf(a) < 1e30f ? (a - f.x) * 2048.0f : 0.0f;
      b = fabsf(b) < 1e30f ? (b - f.y) * 2048.0f : 0.0f;
    }
  }
#pragma unroll
  for (int p = 0; p < P; p++) *reinterpret_cast<uint4*>(at + p * apart) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}

// One CTA per row of x: the row's largest magnitude, and the row in its unit as f16, [part][row], zero from K
// to the padded end.  All ones and nothing: not a row that its unit holds.
template <typename S>
__global__ void __launch_bounds__(512) convert_kernel(const S* __restrict__ x, int64_t K, int64_t ld, int vec, int groups,
                                                      uint8_t* __restrict__ out, uint32_t* __restrict__ top) {
  __shared__ uint32_t most, least;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = blockIdx.x;
  const S* row = x + t * ld;
  auto load = [&](int c, float (&v)[8]) {
    const int64_t left = K - (int64_t)c * 8;
    if (vec && left >= 8) {
      read_x8<S>(reinterpret_cast<const uint8_t*>(row + c * 8), 16, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = e < left ? as_f32(row[c * 8 + e]) : 0.0f;
    }
  };
  if (threadIdx.x == 0) most = 0, least = 0xFFFFFFFFu;
  __syncthreads();
  Range r;
#pragma unroll 4
  for (int c = threadIdx.x; c < groups; c += 512) {
    float v[8];
    load(c, v);
#pragma unroll
    for (int e = 0; e < 8; e++) r.take(v[e]);
  }
  r.top = __reduce_max_sync(0xffffffffu, r.top);
  r.low = __reduce_min_sync(0xffffffffu, r.low);
  if (threadIdx.x % 32 == 0) atomicMax(&most, r.top), atomicMin(&least, r.low);
  __syncthreads();
  const bool fits = in_unit<S>(most, least);
  if (threadIdx.x == 0) top[t] = fits ? most : 0xFFFFFFFFu;
  if (!fits) return;
  const float up = scale_up(most);
#pragma unroll 4
  for (int c = threadIdx.x; c < groups; c += 512) {
    float v[8];
    load(c, v);
    write_x8<S>(out + ((int64_t)t * groups + c) * 16, (int64_t)gridDim.x * groups * 16, v, up);
  }
}

__device__ __forceinline__ void ld_shared(uint32_t at, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
}

// cut_bf16 of finite values.
template <int P> __device__ __forceinline__ void cut_finite(float (&v)[8], uint32_t (&w)[P][4]) {
#pragma unroll
  for (int p = 0; p < P; p++)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      w[p][e / 2] = __byte_perm(__float_as_uint(v[e]), __float_as_uint(v[e + 1]), 0x7632);
      v[e] = __fsub_rn(v[e], __uint_as_float(__float_as_uint(v[e]) & 0xFFFF0000u));
      v[e + 1] = __fsub_rn(v[e + 1], __uint_as_float(__float_as_uint(v[e + 1]) & 0xFFFF0000u));
    }
}

// NB: tiles of eight columns, a column being a part of a token.  DONE: x is what convert_kernel left.
template <int FMT, int NB, typename S, bool DONE>
__global__ void __launch_bounds__(kThreads, 2)
    mx4_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_s,
                      const StreamParams prm, int split) {
  constexpr int P = Parts<S>::k;
  constexpr bool kScaled = Parts<S>::scaled;
  constexpr int kAtoms = FMT == kMXFP4 ? 2 : 4;          // scale tiles of 128 rows x 256 columns
  constexpr int kStage = 128 * 128 + kAtoms * 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int nst = prm.nst;
  const int T = (int)prm.T, cols = T * P;
  // bytes of a column's slice; the odd end keeps eight lanes' 16-byte reads (two columns, four groups) on
  // different banks
  const int xpitch = prm.slice * 2 + 64;
  uint8_t* xs = base + nst * kStage;                     // [part][token] f16 or bf16
  uint32_t* top = reinterpret_cast<uint32_t*>(xs + cols * xpitch);   // largest magnitudes, as bits
  uint32_t* low = top + 16;                              // and one less than the least that are not zero
  uint64_t* bars = reinterpret_cast<uint64_t*>(low + 16);
  volatile int* misc = reinterpret_cast<volatile int*>(bars + 2 * kMaxStages);   // [0] abort, [1] x has an infinity or NaN
  const uint32_t ring = smem_u32(base), full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int tile = (int)blockIdx.x / split;
  const int s_begin = (int)((int64_t)prm.steps * rank / split), s_end = (int)((int64_t)prm.steps * (rank + 1) / split);
  volatile int* abort = &misc[0];

  if (threadIdx.x == 0) {
    for (int s = 0; s < nst; s++) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, kWarps);
    }
    misc[0] = misc[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < 16) top[threadIdx.x] = 0, low[threadIdx.x] = 0xFFFFFFFFu;
  __syncthreads();

  float acc[NB][4];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[b][e] = 0.0f;

  bool fits = true;   // x is held in its rows' units; the same in the whole CTA
  if (warp == kWarps) {
    if (lane == 0) {
      Ring rg{0, 0};
      bool ok = true;
      int loads = 0;
      for (int s = s_begin; s < s_end; s++, loads++) {
        if (loads >= nst && !mbar_wait(empty0 + 8 * rg.st, rg.ph ^ 1, abort, prm.waits.ns)) {
          ok = false;
          break;
        }
        const uint32_t fb = full0 + 8 * rg.st, sw = ring + rg.st * kStage;
        if (loads != prm.waits.skip) {
          mbar_expect_tx(fb, kStage);
          tma_load(sw, &map_w, s * 128, tile * 128, fb);
          tma_load(sw + 128 * 128, &map_s, 0, tile * prm.groups + s * kAtoms, fb);
        }
        rg.advance(nst);
      }
      if (!ok) fail_cta(abort, &g_status);
      for (int k = min(loads, nst); k > 0; k--) {   // every load issued lands before the CTA goes on
        rg.back(nst);
        int zero = 0;
        mbar_wait(full0 + 8 * rg.st, rg.ph, &zero, prm.waits.ns);
      }
    }
  } else {
    // ---- x into shared memory: asynchronous copies of the rows as they are (float32: a group of eight
    // values in its two parts' places), then (scaled types) a pass for their ranges and, if the rows' units hold
    // them, one that converts each group in place.  A warp takes units of 256 columns of one row; a thread
    // reads back only what it copied itself.
    const int units = s_end - s_begin;   // a row's
    const int64_t k0 = (int64_t)s_begin * 256;
    bool odd = false;   // x has an infinity or NaN
    const int apart = T * xpitch;   // from a token's part to its next
    if (DONE) {   // the converted rows are on their way before it is known whether they are there
      asm volatile("griddepcontrol.wait;" ::: "memory");
      for (Unit u(warp, units); u.t < cols; u.next(kWarps, units)) {
        const int c = u.c * 32 + lane;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(xs) + u.t * xpitch + c * 16),
                     "l"(static_cast<const uint8_t*>(prm.units) + u.t * prm.pitch + (k0 / 8 + c) * 16)
                     : "memory");
      }
      const uint32_t m = lane < T ? __ldcg(prm.top + lane) : 0;
      fits = __all_sync(0xffffffffu, m != 0xFFFFFFFFu);
      if (fits) {
        if (warp == 0 && lane < T) top[lane] = m;
      } else {   // another thread may write where this one's copies go
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("bar.sync 1, %0;" ::"r"(32 * kWarps) : "memory");
      }
    }
    if (!(DONE && fits)) {
      constexpr int kChunks = sizeof(S) / 2, kEach = 8 / kChunks;   // of 16 bytes for eight values
      for (Unit u(warp, units); u.t < T; u.next(kWarps, units)) {
        const int c = u.c * 32 + lane;   // group of eight columns
        const int64_t left = prm.K - k0 - (int64_t)c * 8;   // values of the row from here on
        const S* src = static_cast<const S*>(prm.x) + u.t * prm.ld + k0 + c * 8;
        uint8_t* dst = xs + u.t * xpitch + c * 16;
#pragma unroll
        for (int p = 0; p < kChunks; p++) {
          if (prm.vec) {   // sources past the row's end stay at x, which is aligned as its rows are
            const int64_t bytes = (left - p * kEach) * (int64_t)sizeof(S);
            const uint32_t n = bytes >= 16 ? 16 : bytes > 0 ? (uint32_t)bytes : 0;   // the rest is zero
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst) + p * apart),
                         "l"(n ? src + p * kEach : static_cast<const S*>(prm.x)), "r"(n)
                         : "memory");
          } else {
#pragma unroll
            for (int e = 0; e < kEach; e++)
              reinterpret_cast<S*>(dst + p * apart)[e] = p * kEach + e < left ? src[p * kEach + e] : S(0.0f);
          }
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (kScaled && !(DONE && fits)) {   // (what a whole row's unit does not hold, its slice's may)
      bool any = false;
      for (Unit u(warp, units); u.t < T; u.next(kWarps, units)) {
        Range r;
        take_x8<S>(xs + u.t * xpitch + (u.c * 32 + lane) * 16, apart, r);
        r.top = __reduce_max_sync(0xffffffffu, r.top);
        r.low = __reduce_min_sync(0xffffffffu, r.low);
        any |= r.odd;
        if (lane == 0) atomicMax(&top[u.t], r.top), atomicMin(&low[u.t], r.low);
      }
      if (P > 1 && any) misc[1] = 1;
      asm volatile("bar.sync 1, %0;" ::"r"(32 * kWarps) : "memory");
      fits = __all_sync(0xffffffffu, lane >= T || in_unit<S>(top[lane], low[lane]));
      odd = P > 1 && misc[1] != 0;
      if (fits)
        for (Unit u(warp, units); u.t < T; u.next(kWarps, units)) {
          uint8_t* at = xs + u.t * xpitch + (u.c * 32 + lane) * 16;
          float v[8];
          read_x8<S>(at, apart, v);
          write_x8<S>(at, apart, v, scale_up(top[u.t]));
        }
    }
    asm volatile("bar.sync 1, %0;" ::"r"(32 * kWarps) : "memory");

    // ---- the weights
    const int g = lane >> 2, t4 = lane & 3;
    float down[NB][2];   // undoes `up` for this lane's two columns of each tile
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int v = 8 * b + 2 * t4 + e, p = P > 1 && v >= T;
        down[b][e] = kScaled && fits && v < cols ? scale_down(top[v - p * T]) * (p ? 0x1p-11f : 1.0f) : 1.0f;
      }
    const uint32_t row_at = (16 * warp + (lane & 7)) * 128, x7 = lane & 7;
    const uint32_t srow = ((16 * warp + g) & 31) * 16 + ((16 * warp + g) >> 5) * 4;   // row g's scale word; row g + 8: + 128
    // columns past the last read a row that is there; their results are not used
    uint32_t xlane[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) xlane[b] = smem_u32(xs) + (8 * b + g < (fits ? cols : T) ? 8 * b + g : 0) * xpitch + t4 * 16;
    Ring rg{0, 0};
    // EXACT: x as it is, in bf16 (a column is a token; of float32 the three parts one after another); else in its
    // rows' units.  False: a wait ran out.
    auto steps = [&](auto exact) {
      constexpr bool EXACT = decltype(exact)::value;
      constexpr bool kBlocks = !EXACT && FMT == kMXFP4;   // sums of one block
      constexpr int Q = EXACT && P > 1 ? 3 : 1, NBX = EXACT ? (NB + P - 1) / P : NB;
      for (int s = s_begin; s < s_end; s++) {
        if (!mbar_wait_warp(full0 + 8 * rg.st, rg.ph, abort, prm.waits.ns)) return false;
        const uint32_t sw = ring + rg.st * kStage;
        const uint32_t sc = sw + 128 * 128;
        const uint32_t xcol = (s - s_begin) * 512;
        float c[Q][NBX][4];
        if (!kBlocks) {
#pragma unroll
          for (int q = 0; q < Q; q++)
#pragma unroll
            for (int b = 0; b < NBX; b++)
#pragma unroll
              for (int e = 0; e < 4; e++) c[q][b][e] = 0.0f;
        }
#pragma unroll
        for (int half = 0; half < 2; half++) {   // 128 columns
          uint32_t wa[4], wb[4];
          const uint32_t at = sw + row_at + (((half * 4 + (lane >> 3)) ^ x7) << 4);
          ldmatrix4(at, wa);               // rows g: words of four blocks of 32
          ldmatrix4(at + 8 * 128, wb);     // rows g + 8
          uint32_t ha[4], hb[4];           // this lane's scales, twice: bf16 (MXFP4) or f16
          if (FMT == kMXFP4) {
            const uint32_t va = ld_stage_u32(sc + half * 512 + srow);
            const uint32_t vb = ld_stage_u32(sc + half * 512 + srow + 128);
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              const uint32_t a = e8m0x2(va >> (8 * j)), b = e8m0x2(vb >> (8 * j));
              ha[j] = EXACT ? __byte_perm(a, 0, 0x1010) : a << 16, ha[j + 1] = EXACT ? __byte_perm(a, 0, 0x3232) : a & 0xFFFF0000u;
              hb[j] = EXACT ? __byte_perm(b, 0, 0x1010) : b << 16, hb[j + 1] = EXACT ? __byte_perm(b, 0, 0x3232) : b & 0xFFFF0000u;
            }
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
#pragma unroll
            for (int i = 0; i < 4; i++) {
              if (FMT == kNVFP4) a[i] = mul_f16x2(a[i], ha[j]), b[i] = mul_f16x2(b[i], hb[j]);
              if (EXACT) a[i] = f16_to_bf16(a[i]), b[i] = f16_to_bf16(b[i]);
              if (EXACT && FMT == kMXFP4) a[i] = mul_bf16x2(a[i], ha[j]), b[i] = mul_bf16x2(b[i], hb[j]);
            }
#pragma unroll
            for (int nb = 0; nb < NBX; nb++) {
              const uint32_t xat = xlane[nb] + xcol + half * 256 + j * 64;
              uint32_t x[Q][4];
              if constexpr (Q > 1) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 2; e++) ld_shared(xat + e * apart, reinterpret_cast<uint32_t(&)[4]>(v[4 * e]));
                if (odd) cut_bf16<Q>(v, x);
                else cut_finite<Q>(v, x);
              } else {
                ld_shared(xat, x[0]);
              }
              float(&d)[4] = c[0][nb];
              if constexpr (EXACT) {
#pragma unroll
                for (int q = 0; q < Q; q++) {
                  mma_bf16(c[q][nb], a[0], b[0], a[1], b[1], x[q][0], x[q][1]);
                  mma_bf16(c[q][nb], a[2], b[2], a[3], b[3], x[q][2], x[q][3]);
                }
              } else {
                if (kBlocks) mma_f16_zero(d, a[0], b[0], a[1], b[1], x[0][0], x[0][1]);
                else mma_f16(d, a[0], b[0], a[1], b[1], x[0][0], x[0][1]);
                mma_f16(d, a[2], b[2], a[3], b[3], x[0][2], x[0][3]);
              }
              if (kBlocks) {   // two columns at a time, of row g and of row g + 8
#pragma unroll
                for (int r = 0; r < 2; r++) {
                  const float sc8 = __uint_as_float(r ? hb[j] : ha[j]);
                  const float2 v = make_float2(d[2 * r], d[2 * r + 1]);
                  float2* to = reinterpret_cast<float2*>(&acc[nb][2 * r]);
                  *to = __ffma2_rn(kScaled ? __fmul2_rn(v, make_float2(down[nb][0], down[nb][1])) : v, make_float2(sc8, sc8), *to);
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty0 + 8 * rg.st);
        rg.advance(nst);
        if (!kBlocks) {
#pragma unroll
          for (int nb = 0; nb < NBX; nb++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              float v = c[Q - 1][nb][e];   // the smallest part first
#pragma unroll
              for (int q = Q - 2; q >= 0; q--) v += c[q][nb][e];
              acc[nb][e] += EXACT ? v : v * down[nb][e & 1];
            }
        }
      }
      return true;
    };
    const bool ok = !kScaled || fits ? steps(std::false_type{}) : steps(std::true_type{});
    if (!ok) fail_cta(abort, &g_status);
  }
  // ---- results: lane (g, t) has rows g, g + 8 of its warp's 16 and columns 2t, 2t + 1 of each tile
  const int64_t row0 = (int64_t)tile * 128;
  if (split > 1 || P > 1) {
    __syncthreads();   // all loads have landed and been read: the ring is free
    float* part = reinterpret_cast<float*>(base);
    if (warp < kWarps) {
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          // x as it is, of two parts: the columns are tokens and the second parts' are empty
          const int v = 8 * nb + 2 * (lane & 3) + (e & 1), at = 16 * warp + (lane >> 2) + (e >> 1) * 8;
          if (v < cols) part[v * 128 + at] = P == 1 || fits || v < T ? acc[nb][e] : 0.0f;
        }
    }
    if (split > 1) cluster_sync();
    else __syncthreads();
    join_partials<P>(base, rank, split, T, row0, 0, prm.rows, prm.alpha, prm.dtype, prm.y);
    if (split > 1) cluster_sync();
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
  const size_t smem = 1024 + (size_t)p.nst * kStage + (size_t)p.T * Parts<S>::k * (p.slice * 2 + 64) + 128 +
                      16 * kMaxStages + 64;
  return launch_cluster_after<mx4_stream_kernel<FMT, NB, S, DONE>>(DONE, (int)wt * split, kThreads, smem, split, stream, mw,
                                                                  ms, p, split);
}

struct StreamPlan {
  int split, nst, slice;
  bool convert;         // x is converted by a kernel of its own
};
// False where the kernel does not take these sizes: more tokens than it is good for (MXFP4, bf16, here / decoded
// to bf16 for tcgen05: 4096 -> 14336 with 16 tokens 16 / 24 us; a third tile of columns would take 17 tokens at
// 20 / 24 and 24 tokens at 26 / 24), or slices of x that would leave no room in shared memory.
bool stream_plan(int dtype, int64_t T, int64_t rows, int64_t n, StreamPlan* plan) {
  if (T > 16) return false;
  const int64_t wt = (rows + 127) / 128;
  // The converting kernel costs a launch.  4096 -> 14336, with it / without: bf16, 4 tokens 11.9 / 12.1 us, 8
  // tokens 12.3 / 14.3, 16 tokens 16.3 / 22.8; float32, 1 token 12.1 / 11.9, 2 tokens 12.6 / 13.6, 4 tokens 12.8 /
  // 15.9; 4096 -> 4096, bf16, 8 tokens 7.5 / 7.2; float32, 4 tokens 7.7 / 7.7, 12 tokens 11.4 / 13.1.
  const bool convert = dtype != kMxF16 && T * n * wt > (dtype == kMxF32 ? 600000 : 2000000);
  const int parts = dtype == kMxF32 ? Parts<float>::k : 1;
  const int most = 2;   // CTAs to an SM, by registers (three of fewer: one token 4096 -> 14336 12.6 us for 10.3, 16 tokens 24 for 16)
  const int sms = device_sm_count();
  const int steps = (int)(mx4_pitch(n) / 128), stage = 128 * 128 + 4 * 512;   // NVFP4's; MXFP4's is smaller
  int split = 1;
  // one and a half rounds of shorter CTAs beat one of longer ones (14336 -> 4096, bf16: one token 9.6 / 10.6 us, 8
  // tokens 13.0 / 14.1)
  while (split < 8 && wt <= 3 * most / 2 * cluster_slots(split * 2, sms) && split * 2 <= steps) split *= 2;
  // x's slice stays in shared memory beside at least two stages
  auto x_bytes = [&](int sp) { return T * parts * ((int64_t)(steps + sp - 1) / sp * 512 + 64); };
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
  const int64_t cols = p.T * Parts<S>::k;
  if (cols <= 8) return launch_tiles<FMT, 1, S, DONE>(p, w, split, stream);
  if (cols <= 16) return launch_tiles<FMT, 2, S, DONE>(p, w, split, stream);
  if constexpr (Parts<S>::k > 1)
    return cols <= 24 ? launch_tiles<FMT, 3, S, DONE>(p, w, split, stream) : launch_tiles<FMT, 4, S, DONE>(p, w, split, stream);
  return 6;
}

template <int FMT, typename S>
int launch_type(StreamParams& p, const Mx4View& w, int split, bool convert, void* ws, cudaStream_t stream) {
  if constexpr (Parts<S>::scaled) {
    if (convert) {
      const int groups = p.steps * 32;
      p.pitch = (int64_t)groups * 16;
      uint8_t* out = static_cast<uint8_t*>(ws);
      uint32_t* top = reinterpret_cast<uint32_t*>(out + Parts<S>::k * p.T * p.pitch);
      convert_kernel<S><<<(unsigned)p.T, 512, 0, stream>>>(static_cast<const S*>(p.x), p.K, p.ld, p.vec, groups, out, top);
      note_launch();
      p.units = out;
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
  return (size_t)T * (mx4_pitch(n) / 128 * 32 * 16 * (dtype == kMxF32 ? Parts<float>::k : 1) + 4);
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
  p.waits = mx4_take_waits();
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
