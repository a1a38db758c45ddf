// Products with MXFP4 weights for many rows, on the 5th-generation tensor
// cores: y[pair] = W[expert of pair] x[pair] for (row, rank) pairs grouped
// by their expert (a dense product is one expert).
//
// The weights' codes widen to binary16 exactly (fk_mxfp4.cuh), and a power
// of two moves a binary16 within its 40 binades without rounding, so the
// products run as kind::f16 with binary32 accumulators: K moves in runs of
// 512, in each run a weight row's scales are taken relative to the row's
// largest there (2^12 of it; codes of scales 2^36 and more below it lose bits),
// and a row's inputs relative to their largest in the run (2^14 of it). f32
// inputs go as two binary16 parts, x = h1 + h2 within 2^-23 of x or 2^-39 of
// the run's largest, side by side as N columns of one instruction; f16 inputs
// are one part, as they are, and bf16 inputs one, whole down to 2^-31 of the
// run's largest and within 2^-39 of it below. Both factors return when a run's
// sums leave the tensor memory for f32 registers. Runs are short for one more
// reason: the tensor cores cut each accumulation off instead of rounding it. Sums
// of 4096 positive products come out 6.7e-6 of the result too small from the TF32
// GEMM, which adds all of K in place, and 2.3e-7 from the 32 steps of a run here, at
// K = 512 and at 4096.
//
// Three launches:
//   group   the pairs of each expert in order, their slots in expert order, the
//           token tiles of each expert (routed products only);
//   split   a warp a (slot, run): the row's inputs as binary16 parts in
//           slot order, and their factors; pairs without an expert get zeros;
//   tile    persistent CTAs over (expert, token tile, 128 weight rows).
//
// Measured (captured calls): 22016 x 4096 by 511 f32 rows 152 us, 606 TFLOP/s
// (two products each), and 171 us where calls follow one another under the
// power cap, the tensor pipe 61 to 66% busy; by 511 bf16 rows 100 and 111 us; 32000 x 4096
// by 32 bf16 rows 31.8 us; 64 experts of 2816 x 2048, 2048 bf16 rows' 8 each, 266
// and 296 us, of which group 6 and split 15, the tensor pipe 50 to 55% busy. Tiles
// of 64 and fewer tokens are bound by the widening warps (about 2800 cycles a run
// of 512 x 128 weights).
#include <cuda.h>
#include <cudaTypedefs.h>

#include "fk_common.cuh"
#include "fk_kernels.h"
#include "fk_mxfp4.cuh"
#include "fk_tcgen05.cuh"

namespace fk {
namespace lt {

using namespace tc;

constexpr uint32_t kRows = 128;   // weight rows a tile: the MMA's M, TMEM lanes
constexpr uint32_t kSlab = 64;    // K of a slab: 128 bytes of binary16
constexpr uint32_t kRun = 512;    // K of a run
constexpr uint32_t kHalfK = 256;  // K of a stage of codes: 128 bytes, half a run
constexpr uint32_t kSets = 2;                       // of four widening warps, each every other run
constexpr uint32_t kWidenWarps = 4 * kSets;
constexpr uint32_t kInputWarp = 8 + kWidenWarps, kMmaWarp = kInputWarp + 1, kCodeWarp = kInputWarp + 2;
constexpr uint32_t kThreads = 32 * (12 + kWidenWarps);
// Warps: 0..7 drain, then the widening ones, then one that loads inputs, one
// for the MMAs, one that loads codes and one idle. The launch gives each of
// the 640 threads 96 registers (61440 in all); the drain warps, with a
// tile's sums, take 112 and the others 80 (256 x 112 + 384 x 80 = 59392), or
// 128 and 72 (60416) for tiles of 128 and more tokens.
template <int TN>
__device__ __forceinline__ void drain_registers() {
  if constexpr (TN > 96)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
  else
    asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
}
template <int TN>
__device__ __forceinline__ void other_registers() {
  if constexpr (TN > 96)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
}
constexpr uint32_t kMaxSlabs = 16;    // of inputs held: a load takes 1000 to 3000 cycles to land
constexpr uint32_t kCodes = 4;        // stages of codes
constexpr uint32_t kDone = 32;        // steps whose MMAs' end is told apart
constexpr uint32_t kScaleSlots = 12;  // runs whose factors are held
constexpr uint32_t kSmemBudget = 226 * 1024;
constexpr uint32_t kMaxEntries = 4096;

// Status codes (first one wins), after the TF32 GEMMs'.
enum { LT_TIMEOUT_INPUTS = 30, LT_TIMEOUT_CODES = 31, LT_TIMEOUT_WIDEN = 32, LT_TIMEOUT_MMA = 33, LT_TIMEOUT_DRAIN = 34 };

__device__ __forceinline__ void tmem_ld_pair(uint32_t ta, uint32_t tb, uint32_t (&a)[16], uint32_t (&b)[16]) {
  tmem_ld16x2(ta, tb, a, b);
}
__device__ __forceinline__ void tmem_ld_pair(uint32_t ta, uint32_t tb, uint32_t (&a)[8], uint32_t (&b)[8]) {
  tmem_ld8x2(ta, tb, a, b);
}
__device__ __forceinline__ void tmem_ld_one(uint32_t ta, uint32_t (&a)[16]) { tmem_ld16(ta, a); }
__device__ __forceinline__ void tmem_ld_one(uint32_t ta, uint32_t (&a)[8]) { tmem_ld8(ta, a); }

struct Args {
  const uint8_t* scales;
  void* y;
  const uint32_t* perm;  // slot -> pair, or null: the identity
  const uint32_t* off;   // [entries + 1] first slot of each expert, or null: [0, m]
  const uint32_t* tpre;  // [entries + 1] first token tile of each expert
  const float* sx;       // [runs][slots] the inputs' factors
  float* part;           // [2 grid][TN][128] sums of parts of tiles, or null: tiles stay whole
  uint32_t* landed;      // [grid] parts written, of the tile that starts in this CTA
  uint32_t entries, n, kk, k, ldy, slots, wtiles, runs;
};

// Runs r0 .. r1 - 1 of a tile.
struct Piece {
  uint32_t e, slot0, count, row0, r0, r1, tile;
};

// A CTA's work: the tiles' runs in order (or whole tiles), an equal share of
// neighbouring ones each. Experts in order, of an expert the weight tiles in
// order, of a weight tile the token tiles, so that a CTA reads its weights
// from HBM once.
template <int TN>
struct Work {
  uint32_t u, u1, units, per, ctas;  // this CTA's units and all of them, units a tile, CTAs that have any

  __device__ __forceinline__ explicit Work(const Args& a) {
    const uint32_t token_tiles = a.off ? __ldg(a.tpre + a.entries) : (a.slots + TN - 1) / TN;
    per = a.part ? a.runs : 1;
    units = token_tiles * a.wtiles * per;
    ctas = min(gridDim.x, units);
    u = blockIdx.x < ctas ? (uint32_t)((uint64_t)blockIdx.x * units / ctas) : 0;
    u1 = blockIdx.x < ctas ? (uint32_t)((uint64_t)(blockIdx.x + 1) * units / ctas) : 0;
  }
  // The CTA that has unit v.
  __device__ __forceinline__ uint32_t owner(uint32_t v) const {
    return (uint32_t)((((uint64_t)v + 1) * ctas + units - 1) / units - 1);
  }
  __device__ __forceinline__ bool next(const Args& a, Piece& o) {
    if (u >= u1) return false;
    o.tile = u / per;
    o.r0 = a.part ? u - o.tile * per : 0;
    o.r1 = a.part ? min(per, o.r0 + (u1 - u)) : a.runs;
    u += a.part ? o.r1 - o.r0 : 1;
    const uint32_t q = o.tile / a.wtiles;
    uint32_t first = 0, tiles = (a.slots + TN - 1) / TN, s0 = 0, s1 = a.slots;
    o.e = 0;
    if (a.off) {
      uint32_t lo = 0, hi = a.entries;  // the last expert whose first tile is <= q
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (__ldg(a.tpre + mid) <= q)
          lo = mid;
        else
          hi = mid;
      }
      o.e = lo;
      first = __ldg(a.tpre + lo);
      s0 = __ldg(a.off + lo), s1 = __ldg(a.off + lo + 1);
      tiles = __ldg(a.tpre + lo + 1) - first;
    }
    const uint32_t local = o.tile - first * a.wtiles;
    o.slot0 = s0 + (local % tiles) * TN;
    o.count = min((uint32_t)TN, s1 - o.slot0);
    o.row0 = (local / tiles) * kRows;
    return true;
  }
};

// A row's 16 scale bytes of a run, from block b0 on; past the row's nb: 0.
// Rows start on multiples of nb bytes.
__device__ __forceinline__ uint4 load_scales(const uint8_t* row, uint32_t b0, uint32_t nb) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (b0 >= nb) return v;
  if (nb % 16 == 0) return __ldg(reinterpret_cast<const uint4*>(row + b0));
  uint32_t w[4] = {0, 0, 0, 0};
  if (nb % 4 == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (b0 + 4 * i < nb) w[i] = __ldg(reinterpret_cast<const uint32_t*>(row + b0) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (b0 + i < nb) w[i / 4] |= (uint32_t)__ldg(row + b0 + i) << (8 * (i % 4));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// The largest of a run's 16 scale bytes, NaN's (255) left out.
__device__ __forceinline__ uint32_t top_scale(const uint4& s) {
  const uint32_t w[4] = {s.x, s.y, s.z, s.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max_u16x2(m, max_u16x2(w[i] & 0x00FF00FFu, (w[i] >> 8) & 0x00FF00FFu));
  m = max(m & 0xFFFFu, m >> 16);
  if (m == 255) {  // rare
    m = 0;
    for (int i = 0; i < 16; ++i) {
      const uint32_t b = (w[i / 4] >> (8 * (i % 4))) & 0xFFu;
      if (b != 255) m = max(m, b);
    }
  }
  return m;
}

// Slabs a step, of tiles of n columns. A step is what one set of barriers
// stands for: the MMA warp's round of waits and commit takes about 200 cycles
// beside its MMAs, which up to 128 columns take 40 to 64 each, so that two
// slabs share a round there (32000 x 4096 by 32 bf16 rows 35.0 -> 33.2 us, 64
// experts of 2816 x 2048 by 511 x 4 f32 pairs 116 -> 107).
__host__ __device__ constexpr uint32_t step_of(int n) { return n <= 128 ? 2 : 1; }
// All but the inputs' stages: codes, factors, each drain warp's factors
// and output places, barriers, and the alignment's slack.
__host__ __device__ constexpr uint32_t fixed_bytes(int parts, int tn) {
  return kCodes * kRows * 128 + kScaleSlots * kRows * 4 + 8 * (tn / 2) * 12 + 1024 + 1024;
}
__host__ __device__ constexpr uint32_t step_bytes(int parts, int tn) {
  return step_of(parts * tn) * (uint32_t)(parts * tn * 128);
}
__host__ __device__ constexpr uint32_t stages_of(int parts, int tn) {
  const uint32_t fit = (kSmemBudget - fixed_bytes(parts, tn)) / step_bytes(parts, tn);
  return fit < kMaxSlabs / step_of(parts * tn) ? fit : kMaxSlabs / step_of(parts * tn);
}
__host__ __device__ constexpr uint32_t smem_of(int parts, int tn) {
  return fixed_bytes(parts, tn) + stages_of(parts, tn) * step_bytes(parts, tn);
}

template <class E, int PARTS, int TN>
__global__ void __launch_bounds__(kThreads, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, const Args a,
                long long wait_cycles, int* __restrict__ err) {
  constexpr uint32_t N = PARTS * TN;  // the MMA's columns
  constexpr uint32_t P = step_of(N), S = stages_of(PARTS, TN), kCols = 512;
  static_assert(S >= 2, "stages of inputs");
  // Tensor memory: a run's sums, two where they fit, and the widened weights.
  // Each slab of those is 32 columns, each step P slabs.
  constexpr uint32_t kSums = N <= 160 ? 2 : 1, kWide = (N == 160 ? 6 : 8) / P;
  static_assert(kSums * N + 32 * P * kWide <= 512, "tensor memory");
  constexpr uint32_t kHalf = TN / 2;  // a drain warp's tokens
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (an offset, so that the loads stay shared memory's)
  uint8_t* xs = smem;                            // [S][P][N rows][128 bytes]
  uint8_t* raw = xs + S * P * N * 128;               // [kCodes][128 rows][128 bytes]
  uint64_t* places = reinterpret_cast<uint64_t*>(raw + kCodes * kRows * 128);  // [8 drain warps][kHalf]
  float* swb = reinterpret_cast<float*>(places + 8 * kHalf);         // [kScaleSlots][128]
  float* sxb = swb + kScaleSlots * kRows;                            // [8 drain warps][kHalf]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sxb + 8 * kHalf);
  // full: a step's inputs and widened weights; done: its MMAs; rfull and
  // rempty: a stage of codes; afull and aempty: a run's sums; sfull: a run's
  // factors.
  uint64_t *full = bars, *done = full + kDone, *rfull = done + kDone, *rempty = rfull + kCodes,
           *afull = rempty + kCodes, *aempty = afull + 2, *sfull = aempty + 2, *fin = sfull + kScaleSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fin + 1);

  const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t slabs = (a.kk + kSlab - 1) / kSlab;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < kDone; ++s) {
      mbar_init(smem_u32(&full[s]), 5);  // the inputs' loads and a set's four warps
      mbar_init(smem_u32(&done[s]), 1);
    }
    for (uint32_t s = 0; s < kCodes; ++s) {
      mbar_init(smem_u32(&rfull[s]), 1);
      mbar_init(smem_u32(&rempty[s]), 4);  // the warps of the set that widens it
    }
    for (uint32_t s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&afull[s]), 1);
      mbar_init(smem_u32(&aempty[s]), 8);
    }
    for (uint32_t s = 0; s < kScaleSlots; ++s) mbar_init(smem_u32(&sfull[s]), 4);
    mbar_init(smem_u32(fin), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_wait();
  grid_launch_dependents();

  __shared__ uint32_t arrived;
  Work<TN> work(a);
  Piece o;
  // A wait by every lane of a warp, together; false once it ran out.
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
    if (__all_sync(0xffffffffu, mbar_try(smem_u32(bar), parity))) return true;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, wait_cycles));
    if (!ok && lane == 0) record(err, code);
    return ok;
  };
  // The same by one thread.
  auto wait1 = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
    if (mbar_try(smem_u32(bar), parity) || mbar_wait(smem_u32(bar), parity, wait_cycles)) return true;
    record(err, code);
    return false;
  };
  // Step j's MMAs have finished.
  auto done_bar = [&](uint32_t j) { return &done[j % kDone]; };

  if (warp < 8) {
    drain_registers<TN>();
    // Drain: warp w reads TMEM lanes 32 (w % 4).. (weight rows) of the
    // tokens of its half, adds each run's sums, times both factors, and
    // stores a token's 32 neighbouring outputs together.
    const uint32_t quarter = warp & 3, half = warp >> 2;
    float* mysx = sxb + warp * kHalf;
    uint64_t* place = places + warp * kHalf;
    const uint32_t at = tmem + ((32 * quarter) << 16) + half * kHalf;
    uint32_t g = 0;  // runs so far
    bool ok = true;  // false: a wait ran out, the sums are not to be used (the status says so)
    while (work.next(a, o)) {
      float acc[kHalf];
#pragma unroll
      for (uint32_t c = 0; c < kHalf; ++c) acc[c] = 0.0f;
      __syncwarp();
      for (uint32_t c = lane; c < kHalf; c += 32) {
        const uint32_t in_tile = half * kHalf + c, slot = o.slot0 + in_tile;
        const uint32_t p = in_tile >= o.count ? 0 : a.perm ? __ldg(a.perm + slot) : slot;
        place[c] = (uint64_t)(p / a.k) * a.ldy + (uint64_t)(p % a.k) * a.n + o.row0 + 32 * quarter;
      }
      // The tokens' factors of a run are on their way while the run before it
      // is added: looked at below, they would hold up the sums by their latency (64
      // experts of 2816 x 2048 by 2048 x 8 bf16 pairs 298 us so, 266 ahead).
      constexpr uint32_t kOwn = (kHalf + 31) / 32;
      float next[kOwn];
      auto factors = [&](uint32_t run) {
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) {
          const uint32_t c = half * kHalf + lane + 32 * i;
          next[i] = lane + 32 * i < kHalf && c < o.count ? __ldg(a.sx + (size_t)run * a.slots + o.slot0 + c) : 1.0f;
        }
      };
      factors(o.r0);
      for (uint32_t run = o.r0; run < o.r1; ++run, ++g) {
        // The weights' factor and the inputs' are powers of two: their product is
        // exact, or out of binary32's range where a sum times both need not
        // be (weights of 2^-80 by inputs of 2^-60). `within`: no product is,
        // as no weights' factor (2^-104 to 2^115) takes one of 2^-45 to 2^12
        // there. Else the sums take one power after the other, which costs (always:
        // 22016 x 4096 by 511 f32 rows 253 us, 182 so).
        bool within = true;
        __syncwarp();
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) {
          if (lane + 32 * i < kHalf) mysx[lane + 32 * i] = next[i];
          within = within && next[i] >= 0x1p-45f && next[i] <= 0x1p12f;
        }
        within = __all_sync(0xffffffffu, within);
        __syncwarp();
        if (run + 1 < o.r1) factors(run + 1);
        ok = ok && wait(&sfull[g % kScaleSlots], (g / kScaleSlots) & 1, LT_TIMEOUT_WIDEN);
        const float sw = swb[(g % kScaleSlots) * kRows + 32 * quarter + lane];
        if (!within) {  // large inputs, or a run of tiny ones: by the factors themselves
          uint32_t low = __float_as_uint(1.0f), high = low;
          for (uint32_t c = lane; c < kHalf; c += 32)
            low = min(low, __float_as_uint(mysx[c])), high = max(high, __float_as_uint(mysx[c]));
          const float least = __uint_as_float(__reduce_min_sync(0xffffffffu, low));
          const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, high));
          within = __all_sync(0xffffffffu, __fmul_rn(sw, least) > 0.0f && __fmul_rn(sw, most) < INFINITY);
        }
        ok = ok && wait(&afull[g % kSums], g / kSums & 1, LT_TIMEOUT_MMA);
        fence_after();
        const uint32_t from = at + g % kSums * N;
        constexpr uint32_t kPiece = kHalf % 16 ? 8 : 16;
        auto add_run = [&](auto&& add) {
#pragma unroll
          for (uint32_t c = 0; c < kHalf; c += kPiece) {
            uint32_t r0[kPiece];
            [[maybe_unused]] uint32_t r1[kPiece];
            if constexpr (PARTS == 2)
              tmem_ld_pair(from + c, from + TN + c, r0, r1);
            else
              tmem_ld_one(from + c, r0);
#pragma unroll
            for (uint32_t j = 0; j < kPiece; ++j) {
              float v = __uint_as_float(r0[j]);
              if constexpr (PARTS == 2) v = __fadd_rn(v, __uint_as_float(r1[j]));
              acc[c + j] = add(v, mysx[c + j], acc[c + j]);
            }
          }
        };
        if (within)
          add_run([&](float v, float sx, float sum) { return fmaf(v, __fmul_rn(sw, sx), sum); });
        else  // one power after the other
          add_run([&](float v, float sx, float sum) {
            return mx::add_scaled(v, mx::exponent_of(sw) + mx::exponent_of(sx), sum);
          });
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&aempty[g % kSums]));
      }
      if (o.r1 - o.r0 < a.runs) {
        // A part of a tile: its sums to the workspace, by CTA and by whether
        // the tile starts here; the last of the tile's CTAs to do so adds
        // them all, in the CTAs' order.
        constexpr size_t stride = (size_t)TN * kRows;
        constexpr uint32_t kAtOnce = kHalf % 16 ? 8 : 16;
        const uint32_t first = o.tile * a.runs;
        const uint32_t c0 = work.owner(first), c1 = work.owner(first + a.runs - 1);
        const size_t mine = (size_t)(half * kHalf) * kRows + 32 * quarter + lane;
        float* to = a.part + (2 * (size_t)blockIdx.x + (o.r0 == 0 ? 1 : 0)) * stride + mine;
#pragma unroll
        for (uint32_t c = 0; c < kHalf; ++c) to[c * kRows] = acc[c];
        __threadfence();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (threadIdx.x == 0) arrived = atomicAdd(a.landed + c0, 1u);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (arrived != c1 - c0) continue;
        __threadfence();
#pragma unroll
        for (uint32_t c = 0; c < kHalf; ++c) acc[c] = __ldcg(a.part + (2 * (size_t)c0 + 1) * stride + mine + c * kRows);
        for (uint32_t j = c0 + 1; j <= c1; ++j) {
          const float* more = a.part + 2 * (size_t)j * stride + mine;
#pragma unroll
          for (uint32_t c = 0; c < kHalf; c += kAtOnce) {
            float v[kAtOnce];
#pragma unroll
            for (uint32_t d = 0; d < kAtOnce; ++d) v[d] = __ldcg(more + (c + d) * kRows);
#pragma unroll
            for (uint32_t d = 0; d < kAtOnce; ++d) acc[c + d] = __fadd_rn(acc[c + d], v[d]);
          }
        }
      }
      typename E::Storage* y = static_cast<typename E::Storage*>(a.y) + lane;
      // Tokens of this half; none where the lane's row is past the last.
      const uint32_t count = o.row0 + 32 * quarter + lane < a.n ? o.count - min(o.count, half * kHalf) : 0;
#pragma unroll
      for (uint32_t c = 0; c < kHalf; ++c) mx::store_if<E>(c < count, y + place[c], acc[c]);
    }
  } else if (warp < 8 + kWidenWarps) {
    other_registers<TN>();
    // Widen: two sets of four warps, every other run each (a run's scales,
    // factors and waits take a warp as long as half its slabs: in halves of every
    // run 33.1 us for 32000 x 4096 by 32 bf16 rows, so 30.6), a thread a
    // row (its TMEM lane): a slab is 32 bytes of codes (chunk c of row r's 128
    // bytes at c ^ (r % 8), the 128-byte swizzle) to 32 columns of binary16
    // pairs.
    const uint32_t id = threadIdx.x - 256, row = id & 127, set = id >> 7, turn = row & 7;
    const uint32_t nb = a.kk / mx::kBlock;
    const uint8_t* from = raw + row * 128;
    const uint32_t to = tmem + ((32 * (warp & 3)) << 16) + kSums * N;
    uint32_t i0 = 0, g = 0, run = 0;  // steps and runs so far, run of the piece
    auto scales = [&]() {
      return load_scales(a.scales + ((size_t)o.e * a.n + min(o.row0 + row, a.n - 1)) * nb, run * (kRun / mx::kBlock), nb);
    };
    bool ok = true, more = work.next(a, o);
    auto advance = [&]() {
      i0 += (min(slabs - run * (kRun / kSlab), kRun / kSlab) + P - 1) / P;
      ++g;
      if (++run == o.r1 && (more = work.next(a, o))) run = o.r0;
    };
    run = o.r0;
    if (more && set == 1) advance();
    uint4 next = make_uint4(0, 0, 0, 0);
    if (more) next = scales();
    while (ok && more) {
      // A run's scales are loaded while the set's last one is widened.
      const uint4 sc = next;
      const uint32_t at_step = i0, at_run = g, left = slabs - run * (kRun / kSlab);  // slabs of the tile
      advance();
      if (more) advance();
      if (more) next = scales();
      // (Relative to 2^(35 - 127) all codes of smaller scales are binary16 still:
      // rows of zeros, whose scales are 0, have a factor like the others'.)
      const int ref = max((int)top_scale(sc), 35);
      // The factor back: 2^(ref - 127 - 12).
      swb[(at_run % kScaleSlots) * kRows + row] = mx::power_of_two(ref - 139);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sfull[at_run % kScaleSlots]));
      // What takes a scale byte to a binary32 exponent: 2^(byte - ref + 12).
      const int bias = 139 - ref;
#pragma unroll 1
      for (uint32_t half = 0; half < 2; ++half) {
        const uint32_t q = 2 * at_run + half;
        if (!(ok = wait(&rfull[q % kCodes], (q / kCodes) & 1, LT_TIMEOUT_CODES))) break;
        if (4 * half >= left) {  // a stage without codes
          if (lane == 0) mbar_arrive(smem_u32(&rempty[q % kCodes]));
          break;
        }
        const uint32_t mine[2] = {half ? sc.z : sc.x, half ? sc.w : sc.y};  // these eight blocks' scales
        const uint8_t* stage = from + (q % kCodes) * kRows * 128;
        // A step's stores are waited for once a part of the next is widened.
        auto stored = [&](uint32_t i) {
          __syncwarp();
          tmem_wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&full[i % kDone]));
        };
        const uint32_t count = min(left - 4 * half, 4u), first = at_step + 4 / P * half;
#pragma unroll
        for (uint32_t h = 0; h < 4; ++h) {
          if (h >= count) break;
          const uint32_t i = first + h / P, at = to + 32 * (i % kWide * P + h % P);
#pragma unroll
          for (uint32_t c = 0; c < 2; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(stage + (((2 * h + c) ^ turn) << 4));
            const uint32_t byte = (mine[h / 2] >> (16 * (h % 2) + 8 * c)) & 0xFFu;
            // Binary16's own range does the rest: subnormal, then 0.
            const float power = __uint_as_float((uint32_t)max((int)byte + bias, 0) << 23);
            uint32_t by;
            asm("cvt.rn.f16x2.f32 %0, %1, %1;" : "=r"(by) : "f"(byte == 255 ? __uint_as_float(0x7FC00000u) : power));
            const uint32_t words[4] = {v.x, v.y, v.z, v.w};
            uint32_t wide[16];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
              uint32_t f[4];
              mx::widen8_f16(words[u], f);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(wide[4 * u + e]) : "r"(f[e]), "r"(by));
            }
            // Half a slab is widened in registers while the last step's
            // stores are on their way and its columns may be in use.
            if (c == 0 && h % P == 0) {
              if (h > 0) stored(i - 1);
              if (i >= kWide && !(ok = wait(done_bar(i - kWide), (i - kWide) / kDone & 1, LT_TIMEOUT_MMA))) break;
              fence_after();
            }
            __syncwarp();
            tmem_st16(at + 16 * c, wide);
          }
          if (!ok) break;
        }
        if (ok) stored(first + (count - 1) / P);
        if (!ok) break;
        if (lane == 0) mbar_arrive(smem_u32(&rempty[q % kCodes]));
      }
    }
  } else {
  other_registers<TN>();
  if (warp == kInputWarp && elect_one()) {
    // Inputs: a step's slabs of N rows, the parts one below the other.
    uint32_t i = 0, s = 0;
    bool ok = true;
    while (ok && work.next(a, o))
      for (uint32_t slab = o.r0 * (kRun / kSlab), end = min(o.r1 * (kRun / kSlab), slabs); slab < end; slab += P, ++i) {
        if (i >= S && !(ok = wait1(done_bar(i - S), (i - S) / kDone & 1, LT_TIMEOUT_MMA))) break;
        const uint32_t bar = smem_u32(&full[i % kDone]), count = min(end - slab, P);
        mbar_expect_tx(bar, count * N * 128);
        for (uint32_t h = 0; h < count; ++h)
#pragma unroll
          for (int p = 0; p < PARTS; ++p)
            tma_load_3d(smem_u32(xs + (s * P + h) * N * 128 + p * TN * 128), &tx, (int)((slab + h) * kSlab),
                        (int)o.slot0, p, bar);
        s = s + 1 == S ? 0 : s + 1;
      }
    // Loads in flight land before the CTA leaves: the last steps are done
    // (or, where a wait ran out, their bytes have come, within limits).
    for (uint32_t j = i > S ? i - S : 0; j < i; ++j) wait1(&full[j % kDone], j / kDone & 1, LT_TIMEOUT_INPUTS);
  } else if (warp == kCodeWarp && elect_one()) {
    // Codes: half a run a stage, also where a tile's last run has only one.
    uint32_t q = 0;
    bool ok = true;
    while (ok && work.next(a, o))
      for (uint32_t r = o.r0 * (kRun / kHalfK), end = o.r1 * (kRun / kHalfK); r < end; ++r, ++q) {
        const uint32_t s = q % kCodes;
        if (q >= kCodes && !(ok = wait1(&rempty[s], (q / kCodes - 1) & 1, LT_TIMEOUT_WIDEN))) break;
        const uint32_t bar = smem_u32(&rfull[s]);
        if (r * kHalfK < a.kk) {
          mbar_expect_tx(bar, kRows * 128);
          tma_load_3d(smem_u32(raw + s * kRows * 128), &tw, (int)(r * 128), (int)o.row0, (int)o.e, bar);
        } else {
          mbar_arrive(bar);
        }
      }
    for (uint32_t j = q > kCodes ? q - kCodes : 0; j < q; ++j)
      wait1(&rfull[j % kCodes], (j / kCodes) & 1, LT_TIMEOUT_CODES);
  } else if (warp == kMmaWarp && elect_one()) {
    constexpr uint32_t idesc = f16_idesc(N);
    const uint64_t xd0 = sw128_desc(smem_u32(xs));
    uint32_t i = 0, g = 0, s = 0, sw = 0;
    bool ok = true;
    while (ok && work.next(a, o))
      for (uint32_t run = o.r0; ok && run < o.r1; ++run, ++g) {
        if (g >= kSums && !(ok = wait1(&aempty[g % kSums], (g / kSums - 1) & 1, LT_TIMEOUT_DRAIN))) break;
        fence_after();
        const uint32_t to = tmem + g % kSums * N, end = min(kRun / kSlab, slabs - run * (kRun / kSlab));
        for (uint32_t slab = 0; slab < end; slab += P, ++i) {
          if (!(ok = wait1(&full[i % kDone], i / kDone & 1, LT_TIMEOUT_INPUTS))) break;
          fence_after();
          // A K step of 16 is 32 bytes of each row: 2 in a descriptor's address.
          const uint64_t xd = xd0 + s * (P * N * 128 / 16);
          const uint32_t wa = tmem + kSums * N + 32 * P * sw;
#pragma unroll
          for (uint32_t h = 0; h < P; ++h) {
            if (slab + h >= end) break;
#pragma unroll
            for (uint32_t j = 0; j < kSlab / 16; ++j)
              mma_f16_ts(to, wa + 32 * h + 8 * j, xd + h * (N * 128 / 16) + 2 * j, idesc,
                         slab > 0 || h > 0 || j > 0 ? 1u : 0u);
          }
          mma_commit(smem_u32(done_bar(i)));
          s = s + 1 == S ? 0 : s + 1;
          sw = sw + 1 == kWide ? 0 : sw + 1;
        }
        if (ok) mma_commit(smem_u32(&afull[g % kSums]));
      }
    // Every MMA issued has finished before the CTA frees its tensor memory.
    mma_commit(smem_u32(fin));
    wait1(fin, 0, LT_TIMEOUT_MMA);
  }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
}

// ---------------------------------------------------------------------------
// The pairs of each expert

// Gives each expert its run of slots and of token tiles (of tn), and each pair
// a slot of its expert's run, pairs without an expert the last ones. The pairs
// of an expert keep their order: the tile that a pair is in decides where its
// sums are cut, and with that their last bit. A block places `chunk`
// neighbouring pairs (a multiple of 32): it counts all pairs by expert, those
// before its own apart, so that no block waits for another, and one warp goes
// through its own, 32 at a time. (A call of 16000 pairs, 64 experts of 128 x 64:
// 25.8 us; 37.0 by one block with atomics on the experts' next slots, which keep
// no order; 45.6 by one block in order, the warps' counts one after the other.)
__global__ void __launch_bounds__(1024) group_kernel(const uint32_t* __restrict__ ids, uint32_t pairs,
                                                     uint32_t entries, uint32_t tn, uint32_t chunk,
                                                     uint32_t* __restrict__ off, uint32_t* __restrict__ tpre,
                                                     uint32_t* __restrict__ perm, uint32_t* __restrict__ slot_of) {
  __shared__ uint32_t before[kMaxEntries + 1], others[kMaxEntries + 1];  // pairs of each expert (the last: of none)
  __shared__ uint32_t sums[2][32];
  grid_wait();
  grid_launch_dependents();
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, start = blockIdx.x * chunk;
  for (uint32_t e = tid; e <= entries; e += 1024) before[e] = others[e] = 0;
  __syncthreads();
  {
    // Four ids a load, 16 in flight; the last few singly.
    const uint32_t fours = pairs / 4;
    for (uint32_t q0 = tid; q0 < fours; q0 += 4096) {
      uint4 v[4];
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u)
        if (q0 + 1024 * u < fours) v[u] = __ldg(reinterpret_cast<const uint4*>(ids) + q0 + 1024 * u);
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u)
        if (q0 + 1024 * u < fours) {
          uint32_t* count = 4 * (q0 + 1024 * u) < start ? before : others;
          atomicAdd(&count[min(v[u].x, entries)], 1u), atomicAdd(&count[min(v[u].y, entries)], 1u);
          atomicAdd(&count[min(v[u].z, entries)], 1u), atomicAdd(&count[min(v[u].w, entries)], 1u);
        }
    }
    const uint32_t p = 4 * fours + tid;
    if (p < pairs) atomicAdd(&(p < start ? before : others)[min(__ldg(ids + p), entries)], 1u);
  }
  __syncthreads();
  // Thread t has experts 4t .. 4t + 3: exclusive sums of their counts and tiles.
  uint32_t c[4], slots = 0, tiles = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t e = 4 * tid + j;
    c[j] = e < entries ? before[e] + others[e] : 0;
    slots += c[j];
    tiles += (c[j] + tn - 1) / tn;
  }
  uint32_t is = slots, it = tiles;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, is, d), v = __shfl_up_sync(0xffffffffu, it, d);
    if (lane >= (uint32_t)d) is += u, it += v;
  }
  if (lane == 31) sums[0][warp] = is, sums[1][warp] = it;
  __syncthreads();
  if (warp == 0) {
    uint32_t u = sums[0][lane], v = sums[1][lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, u, d), y = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= (uint32_t)d) u += x, v += y;
    }
    sums[0][lane] = u, sums[1][lane] = v;
  }
  __syncthreads();
  uint32_t s = is - slots + (warp ? sums[0][warp - 1] : 0), t = it - tiles + (warp ? sums[1][warp - 1] : 0);
  uint32_t* next = before;  // the expert's next slot of this block
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t e = 4 * tid + j;
    if (e < entries) {
      if (blockIdx.x == 0) off[e] = s, tpre[e] = t;
      next[e] += s;
    }
    s += c[j];
    t += (c[j] + tn - 1) / tn;
  }
  if (tid == 1023) {
    if (blockIdx.x == 0) off[entries] = s, tpre[entries] = t;
    next[entries] += s;
  }
  __syncthreads();
  if (warp != 0) return;
  const uint32_t end = min(pairs, start + chunk);
  constexpr uint32_t kAtOnce = 4;
  for (uint32_t q = start; q < end; q += 32 * kAtOnce) {
    uint32_t e[kAtOnce], alike[kAtOnce];  // a lane's expert, the lanes that have it: they agree in every bit
#pragma unroll
    for (uint32_t u = 0; u < kAtOnce; ++u) {
      const uint32_t p = q + 32 * u + lane;
      e[u] = p < end ? min(__ldg(ids + p), entries) : entries + 1;
      alike[u] = 0xffffffffu;
    }
    for (uint32_t b = 0; (entries + 1) >> b; ++b) {
#pragma unroll
      for (uint32_t u = 0; u < kAtOnce; ++u) {
        const uint32_t set = __ballot_sync(0xffffffffu, e[u] >> b & 1u);
        alike[u] &= e[u] >> b & 1u ? set : ~set;
      }
    }
#pragma unroll
    for (uint32_t u = 0; u < kAtOnce; ++u) {
      const uint32_t p = q + 32 * u + lane;
      const uint32_t slot = p < end ? next[e[u]] + __popc(alike[u] & ((1u << lane) - 1)) : 0;
      __syncwarp();
      if (p < end) {
        if (alike[u] >> lane == 1) next[e[u]] = slot + 1;  // the last of them
        perm[slot] = p;
        slot_of[p] = slot;
      }
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------------------
// The inputs as binary16 parts

struct SplitArgs {
  const void* x;
  void* y;
  uint16_t* parts;  // [PARTS][slots][kk]
  float* sx;        // [runs][slots]
  const uint32_t* slot_of;  // pair -> slot, or null: the identity
  const uint32_t* off;
  uint32_t* landed;  // [grid] set to 0
  uint32_t entries, n, kk, k, ldx, ldy, slots, runs, grid;
  bool per_rank;
};

// A warp a (row or pair with an input of its own, run): 512 inputs, 16 a
// lane, to the slots of all the pairs that take them.
template <class E, int PARTS>
__global__ void __launch_bounds__(256) split_kernel(SplitArgs a) {
  grid_wait();
  grid_launch_dependents();
  const uint32_t lane = threadIdx.x & 31;
  if (blockIdx.x == 0)
    for (uint32_t c = threadIdx.x; c < a.grid; c += 256) a.landed[c] = 0;
  const uint32_t copies = a.per_rank ? 1 : a.k;
  const uint64_t unit = blockIdx.x * 8ull + (threadIdx.x >> 5);
  if (unit >= (uint64_t)(a.slots / copies) * a.runs) return;
  const uint32_t first = (uint32_t)(unit / a.runs) * copies, run = (uint32_t)(unit % a.runs);  // the first pair
  const uint32_t r = first / a.k, j = first % a.k;
  const typename E::Storage* x =
      static_cast<const typename E::Storage*>(a.x) + (size_t)r * a.ldx + (a.per_rank ? (size_t)j * a.kk : 0);
  const bool wide = ((uintptr_t)x & 15) == 0;
  float v[2][8];
  uint32_t top = 0;  // the largest finite magnitude's bits
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t c = run * kRun + 256 * h + 8 * lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[h][i] = 0.0f;
    if (c < a.kk) mx::load8<E>(x, c, wide, v[h]);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, mx::finite_bits(v[h][i]));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  const int up = mx::input_shift<E>(top);
  const float by = mx::scale_value((uint32_t)(127 + up));
  uint32_t lo[2][4], hi[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) mx::split8<PARTS == 2>(v[h], by, hi[h], lo[h]);
  for (uint32_t q = 0; q < copies; ++q) {
    const uint32_t slot = a.slot_of ? __ldg(a.slot_of + first + q) : first + q;
    if (a.off && slot >= __ldg(a.off + a.entries)) {  // a pair without an expert: zeros
      if (run == 0)
        for (uint32_t c = lane; c < a.n; c += 32)
          mx::store<E>(static_cast<typename E::Storage*>(a.y) + (size_t)r * a.ldy + (size_t)(j + q) * a.n + c, 0.0f);
      continue;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t c = run * kRun + 256 * h + 8 * lane;
      if (c >= a.kk) continue;
      uint16_t* to = a.parts + (size_t)slot * a.kk + c;
      *reinterpret_cast<uint4*>(to) = make_uint4(hi[h][0], hi[h][1], hi[h][2], hi[h][3]);
      if constexpr (PARTS == 2)
        *reinterpret_cast<uint4*>(to + (size_t)a.slots * a.kk) = make_uint4(lo[h][0], lo[h][1], lo[h][2], lo[h][3]);
    }
    if (lane == 0) a.sx[(size_t)run * a.slots + slot] = mx::scale_value((uint32_t)(127 - up));
  }
}

}  // namespace lt
}  // namespace fk

namespace {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn_lt() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

// [depth][rows][width] elements as boxes of box_w x box_rows x 1, 128-byte
// swizzle; what lies past any of the three reads as zeros.
bool make_map_lt(CUtensorMap* map, CUtensorMapDataType type, uint32_t elem, const void* base, uint64_t width,
                 uint64_t rows, uint64_t depth, uint32_t box_w, uint32_t box_rows) {
  auto fn = encode_fn_lt();
  if (!fn) return false;
  cuuint64_t dims[3] = {width, rows, depth};
  cuuint64_t strides[2] = {width * elem, width * elem * rows};
  cuuint32_t box[3] = {box_w, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class E, int PARTS, int TN>
cudaError_t launch_tile(const FkLinearMx& a, const fk::lt::Args& g, const uint16_t* parts, uint32_t grid, int* err,
                        bool pdl, cudaStream_t s) {
  using namespace fk::lt;
  constexpr size_t smem = smem_of(PARTS, TN);
  CUtensorMap tx, tw;
  if (!make_map_lt(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, parts, a.kk, g.slots, PARTS, kSlab, TN) ||
      !make_map_lt(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.w, a.kk / 2, a.n, a.entries, kHalfK / 2, kRows))
    return cudaErrorInvalidValue;
  cudaError_t e = fk_allow_smem(tile_kernel<E, PARTS, TN>, smem < 120 * 1024 ? 120 * 1024 : smem);
  if (e != cudaSuccess) return e;
  return fk_launch_ex(tile_kernel<E, PARTS, TN>, dim3(grid), dim3(kThreads),
                      smem < 120 * 1024 ? (size_t)120 * 1024 : smem, s, pdl, tx, tw, g, (long long)4000000000LL, err);
}

// A call's tokens a tile, inputs in so many parts.
uint32_t token_tile(const FkLinearMx& a, int parts, int sms) {
  // The token tile that costs least: the slabs of an SM's tiles, a slab's
  // cost by width, and the last tiles' sums, which nothing covers. Measured,
  // captured, call after call: 22016 x 4096 by 511 rows, f32 in tiles of 16,
  // 32, 64 and 128 tokens 412, 247, 176 and 172 us, bf16 of 16, 32, 64 and 160
  // 404, 216, 133 and 111; 11008 x 4096 by 128 f32 rows, 64 tokens 30 us, 128
  // 35, by 65 rows 30 and 39 (32 tokens 32). Between widths that are even the
  // costs take the wider one, which widens less. Routed experts are uneven:
  // half a tile of each is taken to be empty (64 experts with 32 pairs on
  // average, 2816 x 2048: 32 tokens 123 us, 64 118, 128 185).
  const uint64_t pairs = (uint64_t)a.m * a.k, wtiles = (a.n + fk::lt::kRows - 1) / fk::lt::kRows;
  constexpr uint32_t kWidths = 4;
  const uint32_t widths[kWidths] = {16, 32, 64, parts == 2 ? 128u : 160u};
  const double slab_cost[kWidths] = {100, parts == 2 ? 106. : 104., parts == 2 ? 139. : 114., parts == 2 ? 240. : 151.};
  const double used = pairs < a.entries ? (double)pairs : (double)a.entries;
  const double slabs = used * wtiles * ((a.kk + fk::lt::kSlab - 1) / fk::lt::kSlab) / sms;
  uint32_t tn = 16;
  double least = 0;
  for (uint32_t i = 0; i < kWidths; ++i) {
    const double share = (double)pairs / used / widths[i];
    const double tiles = !a.ids ? (double)((pairs + widths[i] - 1) / widths[i]) : share > 0.5 ? share + 0.5 : 1.0;
    const double cost = tiles * slabs * slab_cost[i] + 70.0 * widths[i];
    if (i == 0 || cost < least) least = cost, tn = widths[i];
  }
  return tn;
}

template <class E, int PARTS>
cudaError_t launch_all(const FkLinearMx& a, int sms, int* err, bool pdl, cudaStream_t s) {
  using namespace fk::lt;
  const uint64_t pairs = (uint64_t)a.m * a.k;
  const uint32_t runs = (a.kk + kRun - 1) / kRun;
  // The workspace: parts, factors, lists, each on a 256-byte boundary.
  uint8_t* at = static_cast<uint8_t*>(a.work);
  auto take = [&](uint64_t bytes) {
    uint8_t* p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  uint16_t* parts = reinterpret_cast<uint16_t*>(take(2 * PARTS * pairs * a.kk));
  float* sx = reinterpret_cast<float*>(take(4 * pairs * runs));
  uint32_t* off = nullptr;
  uint32_t* tpre = nullptr;
  uint32_t* perm = nullptr;
  uint32_t* slot_of = nullptr;
  if (a.ids) {
    off = reinterpret_cast<uint32_t*>(take(4 * (a.entries + 1)));
    tpre = reinterpret_cast<uint32_t*>(take(4 * (a.entries + 1)));
    perm = reinterpret_cast<uint32_t*>(take(4 * pairs));
    slot_of = reinterpret_cast<uint32_t*>(take(4 * pairs));
  }
  const uint32_t tn = token_tile(a, PARTS, sms), wtiles = (a.n + kRows - 1) / kRows;
  if (a.ids) {
    const uint32_t chunk = (uint32_t)((pairs + 32 * sms - 1) / (32 * sms)) * 32;
    cudaError_t e = fk_launch_ex(group_kernel, dim3((uint32_t)((pairs + chunk - 1) / chunk)), dim3(1024), 0, s, pdl,
                                 a.ids, (uint32_t)pairs, a.entries, tn, chunk, off, tpre, perm, slot_of);
    if (e != cudaSuccess) return e;
  }
  // A CTA an SM, each an equal share of the tiles' runs, where the parts of
  // tiles that they leave find room in the workspace; else of whole tiles.
  const uint64_t most =
      (a.ids ? pairs / tn + (pairs < a.entries ? pairs : (uint64_t)a.entries) : (pairs + tn - 1) / tn) * wtiles;  // tiles at most
  uint64_t grid = most < (uint64_t)sms ? most : (uint64_t)sms;
  uint32_t* landed = reinterpret_cast<uint32_t*>(take(4 * (uint64_t)sms));
  const uint64_t left = fk_linear_mxfp4_work(a.entries, a.n, a.kk, a.m, a.k) -
                        (uint64_t)(at - static_cast<uint8_t*>(a.work));
  uint64_t split = most * runs < (uint64_t)sms ? most * runs : (uint64_t)sms;
  if (split * 2 * tn * kRows * 4 > left) split = left / (2 * tn * kRows * 4);
  float* part = nullptr;
  if (split >= grid && runs > 1 && most * runs < 0x80000000ull) {
    grid = split;
    part = reinterpret_cast<float*>(at);
  }
  SplitArgs sp = {a.x,    a.y,   parts, sx,    slot_of, off, landed,          a.entries, a.n,
                  a.kk,   a.k,   a.ldx, a.ldy, (uint32_t)pairs, runs, (uint32_t)grid,  a.per_rank};
  const uint64_t blocks = (pairs / (a.per_rank ? 1 : a.k) * runs + 7) / 8;
  cudaError_t e = fk_launch_ex(split_kernel<E, PARTS>, dim3((uint32_t)blocks), dim3(256), 0, s, pdl, sp);
  if (e != cudaSuccess) return e;
  Args g = {a.scales, a.y, perm, off,   tpre,            sx,     part, landed, a.entries,
            a.n,      a.kk, a.k, a.ldy, (uint32_t)pairs, wtiles, runs};
  const uint32_t ctas = (uint32_t)grid;
  switch (tn) {
    case 16: return launch_tile<E, PARTS, 16>(a, g, parts, ctas, err, pdl, s);
    case 32: return launch_tile<E, PARTS, 32>(a, g, parts, ctas, err, pdl, s);
    case 64: return launch_tile<E, PARTS, 64>(a, g, parts, ctas, err, pdl, s);
    default: return launch_tile<E, PARTS, PARTS == 2 ? 128 : 160>(a, g, parts, ctas, err, pdl, s);
  }
}

}  // namespace

uint32_t fk_linear_mxfp4_tile_tokens(const FkLinearMx& a, FkElem e, int sms) {
  return token_tile(a, e == FK_F32 ? 2 : 1, sms);
}

cudaError_t fk_launch_linear_mxfp4_tile(const FkLinearMx& a, FkElem e, int sms, int* err, bool pdl, cudaStream_t s) {
  if (a.entries > fk::lt::kMaxEntries) return cudaErrorInvalidValue;
  switch (e) {
    case FK_F32: return launch_all<fk::F32, 2>(a, sms, err, pdl, s);
    case FK_BF16: return launch_all<fk::Bf16, 1>(a, sms, err, pdl, s);
    case FK_F16: return launch_all<fk::F16, 1>(a, sms, err, pdl, s);
    default: return cudaErrorInvalidValue;
  }
}
