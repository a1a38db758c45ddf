// Products with MXFP4 weights for many rows, on the 5th-generation tensor
// cores: y[pair] = W[expert of pair] x[pair] for (row, rank) pairs grouped
// by their expert (a dense product is one expert).
//
// The weights' codes widen to binary16 exactly (fk_mxfp4.cuh), and a power
// of two moves a binary16 within its 40 binades without rounding, so the
// products run as kind::f16 with binary32 accumulators: K moves in runs of
// 512, in each run a weight row's scales are taken relative to the row's
// largest there (2^12 of it; a scale more than 2^36 below loses bits of
// values under 2^-36 of the largest), and a row's inputs relative to their
// largest in the run (2^14 of it). f32 inputs go as two binary16 parts, x =
// h1 + h2 within 2^-23 of x or 2^-39 of the run's largest, side by side as
// N columns of one instruction; bf16 and f16 inputs are one part, exact but
// for bf16 values 2^-38 below the run's largest. Both factors return when a
// run's sums leave the tensor memory for f32 registers. Runs are short for
// one more reason: the tensor cores cut each accumulation off instead of
// rounding it, which over all of K = 4096 cost 3xTF32 products 1.4e-5 of
// the result, always toward zero; over the 32 steps of a run it is 5e-7.
//
// Three launches:
//   group   one block: the pairs of each expert, their slots in expert
//           order, the token tiles of each expert (routed products only);
//   split   a warp a (slot, run): the row's inputs as binary16 parts in
//           slot order, and their factors; pairs without an expert get zeros;
//   tile    persistent CTAs over (expert, token tile, 128 weight rows).
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
constexpr uint32_t kSlab = 64;    // K of a stage: 128 bytes of binary16
constexpr uint32_t kRun = 512;    // K of a run
constexpr uint32_t kRawK = 256;   // K of a stage of codes: 128 bytes
constexpr uint32_t kThreads = 608;
// Warps: 0..7 drain, 8..15 widen the weights, 16 loads inputs, 17 the MMAs, 18 loads codes.
constexpr uint32_t kSets = 2;        // of four widening warps, which take slabs in turn
constexpr uint32_t kRawStages = 2;
constexpr uint32_t kWideStages = 3;  // of widened weights
constexpr uint32_t kMaxStages = 6;   // of inputs
constexpr uint32_t kDone = 8;        // slabs whose MMAs' end is told apart
constexpr uint32_t kScaleSlots = 16;
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
  uint32_t entries, n, kk, k, ldy, slots, wtiles;
};

struct Tile {
  uint32_t e, slot0, count, row0;
};

// Tile t: experts in order, of an expert the weight tiles in order, of a
// weight tile the token tiles: CTAs that run together share weights.
template <int TN>
__device__ __forceinline__ bool tile_at(const Args& a, uint32_t t, Tile& o) {
  const uint32_t q = t / a.wtiles;
  uint32_t first = 0, tiles, s0 = 0, s1 = a.slots;
  o.e = 0;
  if (a.off) {
    if (q >= __ldg(a.tpre + a.entries)) return false;
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
  } else {
    tiles = (a.slots + TN - 1) / TN;
    if (q >= tiles) return false;
  }
  const uint32_t local = t - first * a.wtiles;
  o.slot0 = s0 + (local % tiles) * TN;
  o.count = min((uint32_t)TN, s1 - o.slot0);
  o.row0 = (local / tiles) * kRows;
  return true;
}

// Binary16 2^j as a pair, 0 below the type's range.
__device__ __forceinline__ uint32_t half_power2(int j) {
  const uint32_t h = j >= -14 ? (uint32_t)(j + 15) << 10 : j >= -24 ? 1u << (j + 24) : 0u;
  return h | h << 16;
}

// A row's 16 scale bytes of a run, from block b0 on; past the row's nb: 0.
__device__ __forceinline__ uint4 load_scales(const uint8_t* row, uint32_t b0, uint32_t nb) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (b0 >= nb) return v;
  if (nb % 16 == 0 && ((uintptr_t)row & 15) == 0) return __ldg(reinterpret_cast<const uint4*>(row + b0));
  uint32_t w[4] = {0, 0, 0, 0};
  if (nb % 4 == 0 && ((uintptr_t)row & 3) == 0) {
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

// The largest byte of a word, NaN scales (255) left out.
__device__ __forceinline__ uint32_t top_byte(uint32_t w) {
  w &= ~__vcmpeq4(w, 0xFFFFFFFFu);
  w = __vmaxu4(w, w >> 16);
  return max(w & 0xFFu, (w >> 8) & 0xFFu);
}

// All but the inputs' stages: widened weights, codes, factors, each drain
// warp's factors and output places, barriers, and the alignment's slack.
__host__ __device__ constexpr uint32_t fixed_bytes(int tn) {
  return (kWideStages + kRawStages) * kRows * 128 + kScaleSlots * kRows * 4 + 8 * (tn / 2) * 12 + 512 + 1024;
}
__host__ __device__ constexpr uint32_t stages_of(int parts, int tn) {
  return (kSmemBudget - fixed_bytes(tn)) / (uint32_t)(parts * tn * 128) < kMaxStages
             ? (kSmemBudget - fixed_bytes(tn)) / (uint32_t)(parts * tn * 128)
             : kMaxStages;
}
__host__ __device__ constexpr uint32_t smem_of(int parts, int tn) {
  return fixed_bytes(tn) + stages_of(parts, tn) * (uint32_t)(parts * tn * 128);
}

template <class E, int PARTS, int TN>
__global__ void __launch_bounds__(kThreads, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, const Args a,
                long long wait_cycles, int* __restrict__ err) {
  constexpr uint32_t N = PARTS * TN;  // the MMA's columns
  constexpr uint32_t S = stages_of(PARTS, TN);
  constexpr uint32_t kCols = 2 * N < 32 ? 32 : 2 * N;
  constexpr uint32_t kHalf = TN / 2;  // a drain warp's tokens
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (an offset, so that the loads stay shared memory's)
  uint8_t* xs = smem;                            // [S][N rows][128 bytes]
  uint8_t* ws = xs + S * N * 128;                // [kWideStages][128 rows][128 bytes]
  uint8_t* raw = ws + kWideStages * kRows * 128; // [kRawStages][128 rows][128 bytes]
  uint64_t* place = reinterpret_cast<uint64_t*>(raw + kRawStages * kRows * 128);  // [8 drain warps][kHalf]
  float* swb = reinterpret_cast<float*>(place + 8 * kHalf);                      // [kScaleSlots][128]
  float* sxb = swb + kScaleSlots * kRows;                                        // [8 drain warps][kHalf]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sxb + 8 * kHalf);
  // full: a slab's inputs and widened weights; done: its MMAs; rfull and
  // rempty: a stage of codes; afull and aempty: a run's sums; sfull: a run's
  // factors.
  uint64_t *full = bars, *done = full + kDone, *rfull = done + kDone, *rempty = rfull + kRawStages,
           *afull = rempty + kRawStages, *aempty = afull + 2, *sfull = aempty + 2, *fin = sfull + kScaleSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fin + 1);

  const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t slabs = (a.kk + kSlab - 1) / kSlab, runs = (a.kk + kRun - 1) / kRun;
  const uint32_t raws = (a.kk + kRawK - 1) / kRawK;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < kDone; ++s) {
      mbar_init(smem_u32(&full[s]), 5);  // the inputs' loads and a set's four warps
      mbar_init(smem_u32(&done[s]), 1);
    }
    for (uint32_t s = 0; s < kRawStages; ++s) {
      mbar_init(smem_u32(&rfull[s]), 1);
      mbar_init(smem_u32(&rempty[s]), 8);
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
  if (warp == 17) {
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

  Tile o;
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
  // Slab j's MMAs have finished.
  auto done_bar = [&](uint32_t j) { return &done[j % kDone]; };

  if (warp < 8) {
    // Drain: warp w reads TMEM lanes 32 (w % 4).. (weight rows) of the
    // tokens of its half, adds each run's sums, times both factors, and
    // stores a token's 32 neighbouring outputs together.
    const uint32_t quarter = warp & 3, half = warp >> 2;
    float* mysx = sxb + warp * kHalf;
    uint64_t* myplace = place + warp * kHalf;
    const uint32_t at = tmem + ((32 * quarter) << 16) + half * kHalf;
    uint32_t g = 0;  // runs so far
    bool ok = true;
    for (uint32_t t = blockIdx.x; ok && tile_at<TN>(a, t, o); t += gridDim.x) {
      float acc[kHalf];
#pragma unroll
      for (uint32_t c = 0; c < kHalf; ++c) acc[c] = 0.0f;
      __syncwarp();
      for (uint32_t c = lane; c < kHalf; c += 32) {
        const uint32_t slot = o.slot0 + half * kHalf + c;
        if (half * kHalf + c < o.count) {
          const uint32_t p = a.perm ? __ldg(a.perm + slot) : slot;
          myplace[c] = (uint64_t)(p / a.k) * a.ldy + (uint64_t)(p % a.k) * a.n + o.row0 + 32 * quarter;
        }
      }
      for (uint32_t run = 0; run < runs; ++run, ++g) {
        __syncwarp();
        for (uint32_t c = lane; c < kHalf; c += 32)
          mysx[c] = half * kHalf + c < o.count
                        ? __ldg(a.sx + (size_t)run * a.slots + o.slot0 + half * kHalf + c)
                        : 0.0f;
        __syncwarp();
        if (!(ok = wait(&sfull[g % kScaleSlots], (g / kScaleSlots) & 1, LT_TIMEOUT_WIDEN))) break;
        const float sw = swb[(g % kScaleSlots) * kRows + 32 * quarter + lane];
        if (!(ok = wait(&afull[g & 1], (g >> 1) & 1, LT_TIMEOUT_MMA))) break;
        fence_after();
        const uint32_t from = at + (g & 1) * N;
        constexpr uint32_t kPiece = kHalf < 16 ? kHalf : 16;
#pragma unroll
        for (uint32_t c = 0; c < kHalf; c += kPiece) {
          uint32_t r0[kPiece], r1[kPiece];
          if constexpr (PARTS == 2)
            tmem_ld_pair(from + c, from + TN + c, r0, r1);
          else
            tmem_ld_one(from + c, r0);
#pragma unroll
          for (uint32_t j = 0; j < kPiece; ++j) {
            float v = __uint_as_float(r0[j]);
            if constexpr (PARTS == 2) v = __fadd_rn(v, __uint_as_float(r1[j]));
            acc[c + j] = fmaf(v, __fmul_rn(sw, mysx[c + j]), acc[c + j]);
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&aempty[g & 1]));
      }
      if (!ok) break;
      if (o.row0 + 32 * quarter + lane < a.n) {
        typename E::Storage* y = static_cast<typename E::Storage*>(a.y) + lane;
#pragma unroll
        for (uint32_t c = 0; c < kHalf; ++c)
          if (half * kHalf + c < o.count) mx::store<E>(y + myplace[c], acc[c]);
      }
    }
  } else if (warp < 16) {
    // Widen: two sets of four warps take slabs in turn, a thread a row: 32
    // bytes of codes to 128 bytes of binary16, where the 128-byte swizzle
    // puts them (chunk c of row r at c ^ (r % 8)).
    const uint32_t id = threadIdx.x - 256, row = id & 127, set = id >> 7, turn = row & 7;
    const uint32_t nb = a.kk / mx::kBlock;
    const uint8_t* from = raw + row * 128;
    uint8_t* to = ws + row * 128;
    uint32_t i0 = 0, q = 0, g = 0;  // slabs of earlier tiles, code stages, runs so far
    bool ok = true;
    for (uint32_t t = blockIdx.x; ok && tile_at<TN>(a, t, o); t += gridDim.x, i0 += slabs) {
      const uint8_t* srow = a.scales + ((size_t)o.e * a.n + min(o.row0 + row, a.n - 1)) * nb;
      uint4 next = load_scales(srow, 0, nb);
      for (uint32_t run = 0; ok && run < runs; ++run, ++g) {
        const uint4 sc = next;
        next = load_scales(srow, (run + 1) * (kRun / mx::kBlock), nb);
        const int ref = (int)max(max(top_byte(sc.x), top_byte(sc.y)), max(top_byte(sc.z), top_byte(sc.w)));
        if (set == 0) {
          // The factor back: 2^(ref - 127 - 12).
          const int p = ref - 139;
          swb[(g % kScaleSlots) * kRows + row] =
              __uint_as_float(p >= -126 ? (uint32_t)(p + 127) << 23 : 1u << (p + 149));
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sfull[g % kScaleSlots]));
        }
        // The set's half word of scales: blocks 2 slab, 2 slab + 1 of its slabs.
        const uint32_t mine[4] = {sc.x >> (16 * set), sc.y >> (16 * set), sc.z >> (16 * set), sc.w >> (16 * set)};
#pragma unroll
        for (uint32_t j = 0; j < kRun / kSlab / kSets; ++j) {
          const uint32_t slab = run * (kRun / kSlab) + kSets * j + set;
          const uint32_t rs = q % kRawStages;
          const bool staged = slab / 4 * 4 < slabs;  // there is a stage of codes here
          if (j % 2 == 0 && staged && !(ok = wait(&rfull[rs], (q / kRawStages) & 1, LT_TIMEOUT_CODES))) break;
          if (slab < slabs) {
            const uint32_t i = i0 + slab, s = i % kWideStages;
            const uint8_t* cf = from + rs * kRows * 128;
            const uint32_t c = (kSets * j % 4 + set) * 2;  // the slab's first 16 bytes of the stage's 128
            const uint4 c0 = *reinterpret_cast<const uint4*>(cf + ((c ^ turn) << 4));
            const uint4 c1 = *reinterpret_cast<const uint4*>(cf + (((c + 1) ^ turn) << 4));
            uint32_t by[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t byte = (mine[j] >> (8 * h)) & 0xFFu;
              by[h] = byte == 255 ? 0x7E007E00u : half_power2((int)byte - ref + 12);
            }
            if (i >= kWideStages &&
                !(ok = wait(done_bar(i - kWideStages), (i - kWideStages) / kDone & 1, LT_TIMEOUT_MMA)))
              break;
            uint8_t* wt = to + s * kRows * 128;
            const uint32_t words[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
            for (int w = 0; w < 8; ++w) {
              uint32_t h[4];
              mx::widen8_f16(words[w], h);
#pragma unroll
              for (int v = 0; v < 4; ++v) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(h[v]) : "r"(by[w / 4]));
              *reinterpret_cast<uint4*>(wt + ((w ^ turn) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&full[i % kDone]));
          }
          // After a stage of codes: every warp is done with it, those of a set that had none of it too.
          if (j % 2 == 1 && staged) {
            if (lane == 0) mbar_arrive(smem_u32(&rempty[rs]));
            ++q;
          }
        }
      }
    }
  } else if (warp == 16 && elect_one()) {
    // Inputs: a slab's N rows, the parts one below the other.
    uint32_t i = 0, s = 0;
    bool ok = true;
    for (uint32_t t = blockIdx.x; ok && tile_at<TN>(a, t, o); t += gridDim.x)
      for (uint32_t slab = 0; slab < slabs; ++slab, ++i) {
        if (i >= S && !(ok = wait1(done_bar(i - S), (i - S) / kDone & 1, LT_TIMEOUT_MMA))) break;
        const uint32_t bar = smem_u32(&full[i % kDone]);
        mbar_expect_tx(bar, N * 128);
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
          tma_load_3d(smem_u32(xs + s * N * 128 + p * TN * 128), &tx, (int)(slab * kSlab), (int)o.slot0, p, bar);
        s = s + 1 == S ? 0 : s + 1;
      }
    // Loads in flight land before the CTA leaves: the last slabs are done
    // (or, where a wait ran out, their bytes have come, within limits).
    for (uint32_t j = i > S ? i - S : 0; j < i; ++j) wait1(&full[j % kDone], j / kDone & 1, LT_TIMEOUT_INPUTS);
  } else if (warp == 18 && elect_one()) {
    // Codes: 256 of K a stage.
    uint32_t q = 0;
    bool ok = true;
    for (uint32_t t = blockIdx.x; ok && tile_at<TN>(a, t, o); t += gridDim.x)
      for (uint32_t r = 0; r < raws; ++r, ++q) {
        const uint32_t s = q % kRawStages;
        if (q >= kRawStages && !(ok = wait1(&rempty[s], (q / kRawStages - 1) & 1, LT_TIMEOUT_WIDEN))) break;
        const uint32_t bar = smem_u32(&rfull[s]);
        mbar_expect_tx(bar, kRows * 128);
        tma_load_3d(smem_u32(raw + s * kRows * 128), &tw, (int)(r * 128), (int)o.row0, (int)o.e, bar);
      }
    for (uint32_t j = q > kRawStages ? q - kRawStages : 0; j < q; ++j)
      wait1(&rfull[j % kRawStages], (j / kRawStages) & 1, LT_TIMEOUT_CODES);
  } else if (warp == 17 && elect_one()) {
    constexpr uint32_t idesc = f16_idesc(N);
    const uint64_t wd0 = sw128_desc(smem_u32(ws)), xd0 = sw128_desc(smem_u32(xs));
    uint32_t i = 0, g = 0, s = 0, sw = 0;
    bool ok = true;
    for (uint32_t t = blockIdx.x; ok && tile_at<TN>(a, t, o); t += gridDim.x)
      for (uint32_t run = 0; ok && run < runs; ++run, ++g) {
        if (g >= 2 && !(ok = wait1(&aempty[g & 1], ((g >> 1) - 1) & 1, LT_TIMEOUT_DRAIN))) break;
        fence_after();
        const uint32_t to = tmem + (g & 1) * N, end = min(kRun / kSlab, slabs - run * (kRun / kSlab));
        for (uint32_t slab = 0; slab < end; ++slab, ++i) {
          if (!(ok = wait1(&full[i % kDone], i / kDone & 1, LT_TIMEOUT_INPUTS))) break;
          fence_after();
          // A K step of 16 is 32 bytes of each row: 2 in a descriptor's address.
          const uint64_t wd = wd0 + sw * (kRows * 128 / 16), xd = xd0 + s * (N * 128 / 16);
#pragma unroll
          for (uint32_t j = 0; j < kSlab / 16; ++j)
            mma_f16(to, wd + 2 * j, xd + 2 * j, idesc, slab > 0 || j > 0 ? 1u : 0u);
          mma_commit(smem_u32(done_bar(i)));
          s = s + 1 == S ? 0 : s + 1;
          sw = sw + 1 == kWideStages ? 0 : sw + 1;
        }
        if (ok) mma_commit(smem_u32(&afull[g & 1]));
      }
    // Every MMA issued has finished before the CTA frees its tensor memory.
    mma_commit(smem_u32(fin));
    wait1(fin, 0, LT_TIMEOUT_MMA);
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 17)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
}

// ---------------------------------------------------------------------------
// The pairs of each expert

// One block. Counts the experts' pairs, gives each expert its run of slots
// and of token tiles (of tn), and each pair a slot of its expert's run, pairs
// without an expert the last ones. Which slot of the run a pair gets depends
// on the order in which the atomics land; no result does, since a token's
// column of a tile is computed by itself.
__global__ void __launch_bounds__(1024) group_kernel(const uint32_t* __restrict__ ids, uint32_t pairs,
                                                     uint32_t entries, uint32_t tn, uint32_t* __restrict__ off,
                                                     uint32_t* __restrict__ tpre, uint32_t* __restrict__ perm) {
  __shared__ uint32_t count[kMaxEntries];
  __shared__ uint32_t sums[2][32];
  __shared__ uint32_t rest;
  grid_wait();
  grid_launch_dependents();
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (uint32_t e = tid; e < kMaxEntries; e += 1024) count[e] = 0;
  __syncthreads();
  for (uint32_t p = tid; p < pairs; p += 1024) {
    const uint32_t e = __ldg(ids + p);
    if (e < entries) atomicAdd(&count[e], 1u);
  }
  __syncthreads();
  // Thread t has experts 4t .. 4t + 3: exclusive sums of their counts and tiles.
  uint32_t c[4], slots = 0, tiles = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    c[j] = count[4 * tid + j];
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
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t e = 4 * tid + j;
    if (e < entries) off[e] = s, tpre[e] = t;
    count[e] = s;  // the expert's next slot
    s += c[j];
    t += (c[j] + tn - 1) / tn;
  }
  if (tid == 1023) {
    off[entries] = s;
    tpre[entries] = t;
    rest = s;
  }
  __syncthreads();
  for (uint32_t p = tid; p < pairs; p += 1024) {
    const uint32_t e = __ldg(ids + p);
    perm[e < entries ? atomicAdd(&count[e], 1u) : atomicAdd(&rest, 1u)] = p;
  }
}

// ---------------------------------------------------------------------------
// The inputs as binary16 parts

struct SplitArgs {
  const void* x;
  void* y;
  uint16_t* parts;  // [PARTS][slots][kk]
  float* sx;        // [runs][slots]
  const uint32_t* perm;
  const uint32_t* off;
  uint32_t entries, n, kk, k, ldx, ldy, slots, runs;
  bool per_rank;
};

// A warp a (slot, run): 512 inputs, 16 a lane.
template <class E, int PARTS>
__global__ void __launch_bounds__(256) split_kernel(SplitArgs a) {
  grid_wait();
  grid_launch_dependents();
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t unit = blockIdx.x * 8ull + (threadIdx.x >> 5);
  if (unit >= (uint64_t)a.slots * a.runs) return;
  const uint32_t slot = (uint32_t)(unit / a.runs), run = (uint32_t)(unit % a.runs);
  const uint32_t p = a.perm ? __ldg(a.perm + slot) : slot;
  const uint32_t r = p / a.k, j = p % a.k;
  if (a.off && slot >= __ldg(a.off + a.entries)) {  // a pair without an expert
    if (run == 0)
      for (uint32_t c = lane; c < a.n; c += 32)
        mx::store<E>(static_cast<typename E::Storage*>(a.y) + (size_t)r * a.ldy + (size_t)j * a.n + c, 0.0f);
    return;
  }
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
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t c = run * kRun + 256 * h + 8 * lane;
    if (c >= a.kk) continue;
    uint32_t lo[4], hi[4];
    mx::split8<PARTS == 2>(v[h], by, hi, lo);
    uint16_t* to = a.parts + (size_t)slot * a.kk + c;
    *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if constexpr (PARTS == 2)
      *reinterpret_cast<uint4*>(to + (size_t)a.slots * a.kk) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
  if (lane == 0) a.sx[(size_t)run * a.slots + slot] = mx::scale_value((uint32_t)(127 - up));
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
cudaError_t launch_tile(const FkLinearMx& a, const fk::lt::Args& g, const uint16_t* parts, uint64_t most, int sms,
                        int* err, bool pdl, cudaStream_t s) {
  using namespace fk::lt;
  constexpr size_t smem = smem_of(PARTS, TN);
  CUtensorMap tx, tw;
  if (!make_map_lt(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, parts, a.kk, g.slots, PARTS, kSlab, TN) ||
      !make_map_lt(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.w, a.kk / 2, a.n, a.entries, 128, kRows))
    return cudaErrorInvalidValue;
  cudaError_t e = fk_allow_smem(tile_kernel<E, PARTS, TN>, smem < 120 * 1024 ? 120 * 1024 : smem);
  if (e != cudaSuccess) return e;
  const uint64_t grid = most < (uint64_t)sms ? most : (uint64_t)sms;
  return fk_launch_ex(tile_kernel<E, PARTS, TN>, dim3((uint32_t)grid), dim3(kThreads),
                      smem < 120 * 1024 ? (size_t)120 * 1024 : smem, s, pdl, tx, tw, g, (long long)4000000000LL, err);
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
  if (a.ids) {
    off = reinterpret_cast<uint32_t*>(take(4 * (a.entries + 1)));
    tpre = reinterpret_cast<uint32_t*>(take(4 * (a.entries + 1)));
    perm = reinterpret_cast<uint32_t*>(take(4 * pairs));
  }
  // Token tiles as wide as an expert's mean share asks for.
  const uint64_t share = (pairs + a.entries - 1) / a.entries;
  const uint32_t tn = share <= 16 ? 16 : share <= 32 ? 32 : share <= 64 ? 64 : 128;
  if (a.ids) {
    cudaError_t e = fk_launch_ex(group_kernel, dim3(1), dim3(1024), 0, s, pdl, a.ids, (uint32_t)pairs, a.entries, tn,
                                 off, tpre, perm);
    if (e != cudaSuccess) return e;
  }
  SplitArgs sp = {a.x, a.y, parts, sx, perm, off, a.entries, a.n, a.kk, a.k, a.ldx, a.ldy, (uint32_t)pairs, runs,
                  a.per_rank};
  const uint64_t blocks = (pairs * runs + 7) / 8;
  cudaError_t e = fk_launch_ex(split_kernel<E, PARTS>, dim3((uint32_t)blocks), dim3(256), 0, s, pdl, sp);
  if (e != cudaSuccess) return e;
  Args g = {a.scales, a.y, perm, off, tpre, sx, a.entries, a.n, a.kk, a.k, a.ldy, (uint32_t)pairs,
            (a.n + kRows - 1) / kRows};
  const uint64_t most =
      (pairs / tn + (a.ids ? (pairs < a.entries ? pairs : (uint64_t)a.entries) : 1)) * g.wtiles;  // tiles at most
  if (tn == 16) return launch_tile<E, PARTS, 16>(a, g, parts, most, sms, err, pdl, s);
  if (tn == 32) return launch_tile<E, PARTS, 32>(a, g, parts, most, sms, err, pdl, s);
  if (tn == 64) return launch_tile<E, PARTS, 64>(a, g, parts, most, sms, err, pdl, s);
  return launch_tile<E, PARTS, 128>(a, g, parts, most, sms, err, pdl, s);
}

}  // namespace

cudaError_t fk_launch_linear_mxfp4_tile(const FkLinearMx& a, FkElem e, int sms, int* err, bool pdl, cudaStream_t s) {
  if (a.entries > fk::lt::kMaxEntries) return cudaErrorInvalidValue;
  switch (e) {
    case FK_F32: return launch_all<fk::F32, 2>(a, sms, err, pdl, s);
    case FK_BF16: return launch_all<fk::Bf16, 1>(a, sms, err, pdl, s);
    case FK_F16: return launch_all<fk::F16, 1>(a, sms, err, pdl, s);
    default: return cudaErrorInvalidValue;
  }
}
