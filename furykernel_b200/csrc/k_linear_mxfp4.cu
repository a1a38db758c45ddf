// Products with MXFP4 weights (fk_mxfp4.cuh): y[r, j] = W[ids[r, j]] x[r],
// or x[r, j] where each rank has its own input; a dense product is one
// expert that every row takes. x and y in f32, bf16 or f16; the products
// and sums in binary32, the result rounded once. Two kernels: the streaming
// one below for few rows an expert, the tcgen05 one
// (k_linear_mxfp4_tile.cu) for more.
//
// The streaming kernel reads every weight once for up to R rows and should
// be held by HBM, so the arithmetic a weight has to be little: at 23 bytes
// (43 weights) a cycle an SM there are three instructions a weight, and one
// and a half of the integer pipe's, which also widens codes. The codes go,
// widened two an instruction to binary16 and unscaled, to the tensor cores'
// warp-wide products (16 weight rows x 16 of K x 8 columns); a block of 32
// weights, two such products, is one scale, which multiplies the block's
// sums. The columns are the inputs: a row as two binary16 parts, x = h1 +
// h2 relative to the largest of a stage's 256 (within 2^-23 of x or 2^-39
// of that largest), so 8 columns are 4 rows. Sums of blocks are binary32;
// rows with scales of 2^65 and more, which could take them out of its
// range before the inputs' power is back, are summed a second time.
//
// Measured (captured launches over weights that are not in L2): 32000 x 4096
// by one f32 row 20.6 us, 3.4 TB/s of codes and scales, by 4 rows 25.2 us; 64
// experts of 2816 x 2048, 8 rows' 8 experts each, 37 us, 3.4 TB/s; 1408 x 2048
// by one row's 4 experts 7.0 us. A launch, the inputs' splitting and the first
// stages are 5 to 6 us of each; past them 4.4 TB/s, with the SMs issuing in
// half of their cycles and the warps at each other's sums.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "fk_common.cuh"
#include "fk_kernels.h"
#include "fk_mxfp4.cuh"
#include "fk_tcgen05.cuh"

namespace fk {
namespace ls {

using namespace tc;

constexpr uint32_t kWarps = 16;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr uint32_t kTileRows = 16;     // weight rows of a unit
constexpr uint32_t kStageBlocks = 8;   // blocks of 32 weights a row a stage: 128 bytes of codes
constexpr uint32_t kCodeBytes = kTileRows * kStageBlocks * 16;
constexpr uint32_t kScaleWords = 3;    // the words that hold 8 bytes, wherever they start
constexpr uint32_t kMaxPairs = 512;
constexpr uint32_t kBatch = 8, kLeastBatch = 4;  // units whose sums wait together: at best, where shared memory is short
constexpr uint32_t kMaxEntries = 4096;
constexpr uint32_t kSmemBudget = 227 * 1024 - 1024;  // static and dynamic, less the alignment's slack

enum { LS_TIMEOUT = 29 };  // a stage of codes never landed

// Stages of a warp's own ring.
constexpr uint32_t kStages = 3;

// What the weights' factors are moved up by, in binades (the smallest scales'
// products with small inputs keep their bits so); the inputs' take it back.
constexpr int kMoved = 16;
// A stage's scale words and their values as factors.
constexpr uint32_t kScaleBytes = kTileRows * kScaleWords * 4;
constexpr uint32_t kFactorBytes = kTileRows * kStageBlocks * 4;

// A group's inputs: `steps` stages of R rows, two parts of 512 bytes each,
// and a factor a row and stage.
__host__ __device__ constexpr uint32_t input_bytes(uint32_t steps, uint32_t R) {
  return steps * R * kStageBlocks * 128 + (steps * R * 4 + 15) / 16 * 16;
}
// A warp's scale words and factors, and all of a block's shared memory.
constexpr uint32_t kOwnBytes = kStages * kScaleBytes + kFactorBytes;
// Units whose sums wait together: `batch` of them.
__host__ __device__ constexpr uint32_t sum_bytes(uint32_t batch, uint32_t R) {
  return batch * kWarps * kTileRows * R * 4;
}
__host__ __device__ constexpr uint32_t block_bytes(uint32_t steps, uint32_t share, uint32_t batch, uint32_t R) {
  return kWarps * (kStages * kCodeBytes + kOwnBytes) + kWarps / share * input_bytes(steps, R) + sum_bytes(batch, R);
}
constexpr uint32_t kStaticBytes = kMaxPairs * 12 + kThreads * 4 + 1024 + kWarps * kStages * 8;

// Four bytes, of which `have` are there (the others become 0).
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, uint32_t have) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(have) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same onto zeros.
__device__ __forceinline__ void mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// One block of 32: two products of the codes of rows g and g + 8 (four bytes a
// lane of each) with the inputs' parts, and the rows' sums.
__device__ __forceinline__ void block_sums(uint32_t codes0, uint32_t codes1, const uint4& x, float& v0, float& v1) {
  uint32_t p[4], q[4];
  mx::widen8_f16(codes0, p);
  mx::widen8_f16(codes1, q);
  float d[4];
  mma0(d, p[0], q[0], p[1], q[1], x.x, x.y);
  mma(d, p[2], q[2], p[3], q[3], x.z, x.w);
  v0 = __fadd_rn(d[0], d[1]), v1 = __fadd_rn(d[2], d[3]);
}

// Scale bytes from here on (2^65) may take sums of inputs that were moved up
// out of binary32's range; 255 is no power.
constexpr uint32_t kLarge = 192;

// A warp's sums of a unit once more, from global memory, for its rows with
// large scales: a block's sum takes its own power and the inputs' at once.
// `codes`, `scales`: row g's, of `blocks` blocks, row g + 8 eight rows on; the
// warp's blocks are b0 .. b1 - 1, its inputs at xat and sat, its sums at to[0]
// and to[8] (of lanes that have any).
__device__ __forceinline__ void sum_large(const uint8_t* codes, const uint8_t* scales, uint32_t blocks, uint32_t b0,
                                          uint32_t b1, const uint4* xat, const float* sat, uint32_t R, bool any,
                                          float* to) {
  float acc[2] = {0.0f, 0.0f};
  uint32_t top[2] = {0, 0};
#pragma unroll 1
  for (uint32_t b = b0; b < b1; ++b, xat += 8 * R) {
    float v[2];
    block_sums(__ldg(reinterpret_cast<const uint32_t*>(codes + 16ull * b)),
               __ldg(reinterpret_cast<const uint32_t*>(codes + 16 * (b + 8ull * blocks))), *xat, v[0], v[1]);
    const int up = mx::exponent_of(sat[(b - b0) / kStageBlocks * R]) + kMoved - 127;
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t s = __ldg(scales + b + 8ull * h * blocks);
      acc[h] = s == 255 ? __uint_as_float(0x7FC00000u) : mx::add_scaled(v[h], (int)s + up, acc[h]);
      top[h] = max(top[h], s);
    }
  }
  if (any && top[0] >= kLarge) to[0] = acc[0];
  if (any && top[1] >= kLarge) to[8] = acc[1];
}

// A pass: up to R pairs of one expert, at `first` of the grouped pairs.
struct Pass {
  uint16_t first, count;
  uint32_t e;
};

// Persistent blocks over units (pass, 16 weight rows). A group of `share`
// warps takes neighbouring units; its warps split a unit's K, each with
// its own ring of stages, so that a warp's loads run on over the units, and
// its own part of the inputs, so that only the unit's last sum needs the
// others.
template <class E, int R>
__global__ void __launch_bounds__(kThreads, 1)
    stream_kernel(const __grid_constant__ CUtensorMap tw, const FkLinearMx a, uint32_t share, uint32_t batch,
                  long long wait_cycles, int* __restrict__ err) {
  constexpr uint32_t stages = kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t landed[kWarps][stages];
  __shared__ Pass passes[kMaxPairs];
  __shared__ uint32_t perm[kMaxPairs];  // a pair's row, its rank << 16
  __shared__ uint32_t ids_s[kThreads];
  __shared__ uint32_t sums[2][kWarps], npasses_s, nrest_s;
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (an offset, so that the loads stay shared memory's)
  const uint32_t blocks = a.kk / mx::kBlock, all_steps = (blocks + kStageBlocks - 1) / kStageBlocks;
  // [kWarps][stages] codes, each warp's scale words and factors, each group's inputs,
  // [batch][kWarps][R][16] sums.
  uint8_t* rest_smem = smem + kWarps * stages * kCodeBytes;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t pairs = a.m * a.k, tiles = (a.n + kTileRows - 1) / kTileRows;

  // The weights too may be the previous launch's (quant_mxfp4's): nothing is read before it is done.
  if (tid < kWarps * stages) mbar_init(smem_u32(&landed[0][0] + tid), 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  grid_wait();
  grid_launch_dependents();
  uint32_t npasses, rest = 0;
  if (a.ids) {
    // The pairs of each expert, in the input's space (not filled yet).
    uint32_t* count = reinterpret_cast<uint32_t*>(rest_smem);
    const uint32_t most = (a.entries + kThreads - 1) / kThreads;  // experts a thread, at most 8
    for (uint32_t e = tid; e < most * kThreads; e += kThreads) count[e] = 0;
    // A pair's expert (entries: none) and its place among the expert's pairs,
    // by index: every block has to list them alike.
    const uint32_t own = tid < pairs ? min(__ldg(a.ids + tid), a.entries) : 0xffffffffu;
    ids_s[tid] = own;
    __syncthreads();
    uint32_t place = 0;
    if (own < a.entries) atomicAdd(&count[own], 1u);
    for (uint32_t q = 0; q < (tid & ~31u) + 32 && q < pairs; ++q) place += q < tid && ids_s[q] == own;
    __syncthreads();
    uint32_t c[8], mine = 0, mypass = 0;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      c[j] = j < most ? count[tid * most + j] : 0u;
      mine += c[j];
      mypass += (c[j] + R - 1) / R;
    }
    uint32_t is = mine, ip = mypass;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, is, d), v = __shfl_up_sync(0xffffffffu, ip, d);
      if (lane >= (uint32_t)d) is += u, ip += v;
    }
    if (lane == 31) sums[0][warp] = is, sums[1][warp] = ip;
    __syncthreads();
    uint32_t bs = 0, bp = 0;
    for (uint32_t w = 0; w < warp; ++w) bs += sums[0][w], bp += sums[1][w];
    uint32_t s = bs + is - mine, p = bp + ip - mypass;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      if (j >= most) break;
      count[tid * most + j] = s;
      for (uint32_t q = 0; q < c[j]; q += R) {
        passes[p].first = (uint16_t)(s + q);
        passes[p].count = (uint16_t)min((uint32_t)R, c[j] - q);
        passes[p].e = tid * most + j;
        ++p;
      }
      s += c[j];
    }
    if (tid == kThreads - 1) npasses_s = p, nrest_s = s;
    __syncthreads();
    npasses = npasses_s;
    rest = nrest_s;
    if (tid < pairs) perm[(own < a.entries ? count[own] : rest) + place] = tid / a.k | (tid % a.k) << 16;
    __syncthreads();
    // Pairs without an expert: zeros.
    for (uint32_t q = rest + blockIdx.x; q < pairs; q += gridDim.x)
      for (uint32_t i = tid; i < a.n; i += kThreads)
        mx::store<E>(static_cast<typename E::Storage*>(a.y) + (size_t)(perm[q] & 0xFFFFu) * a.ldy +
                         (size_t)(perm[q] >> 16) * a.n + i,
                     0.0f);
  } else {
    npasses = (pairs + R - 1) / R;
    if (tid < npasses) {
      passes[tid].first = (uint16_t)(tid * R);
      passes[tid].count = (uint16_t)min((uint32_t)R, pairs - tid * R);
      passes[tid].e = 0;
    }
    if (tid < pairs) perm[tid] = tid / a.k | (tid % a.k) << 16;
    __syncthreads();
  }

  const uint32_t abreast = kWarps / share, group = warp / share, part = warp % share;
  const uint64_t units = (uint64_t)npasses * tiles, groups = (uint64_t)gridDim.x * abreast,
                 gid = (uint64_t)blockIdx.x * abreast + group;
  const uint32_t u0 = (uint32_t)(gid * units / groups), u1 = (uint32_t)((gid + 1) * units / groups);
  // This warp's stages of every row.
  const uint32_t s0 = part * all_steps / share, steps = (part + 1) * all_steps / share - s0;
  const uint64_t scale_bytes = (uint64_t)a.entries * a.n * blocks;
  const uint32_t ring = smem_u32(smem) + warp * stages * kCodeBytes;
  uint8_t* mine_smem = rest_smem + warp * kOwnBytes;
  const uint32_t scale_ring = smem_u32(mine_smem);
  float* factors = reinterpret_cast<float*>(mine_smem + stages * kScaleBytes);  // [16 rows][8]
  // The inputs, [blocks][R][4][2] 16 bytes as the products take them, and
  // the factors back, [steps][R]: this warp's of its group's.
  uint8_t* group_smem = rest_smem + kWarps * kOwnBytes + group * input_bytes(all_steps, R);
  auto red = reinterpret_cast<float(*)[kWarps][kTileRows * R]>(rest_smem + kWarps * kOwnBytes +
                                                               abreast * input_bytes(all_steps, R));
  uint8_t* xs = group_smem + s0 * kStageBlocks * R * 128;
  float* sxs = reinterpret_cast<float*>(group_smem + all_steps * kStageBlocks * R * 128) + s0 * R;

  // A unit's first row, and where this warp's scale bytes of row `of` of it
  // start. A unit's rows end with the table's: the last unit starts early
  // enough (its first rows are another's too, with the same results).
  auto first_row = [&](uint32_t tile) { return min(tile * kTileRows, a.n - kTileRows); };
  auto first_scale = [&](uint32_t pass, uint32_t tile, uint32_t of) {
    return ((uint64_t)passes[pass].e * a.n + first_row(tile) + of) * blocks + s0 * kStageBlocks;
  };

  // The loads of the next stage: the warp's own cursor over (unit, step). A
  // lane's scale word is word lane % 2 of the row's (the even lanes take
  // word 2 too, where the bytes reach into it); the table's last word may
  // be short. From one unit to the next of a pass all of it moves on by 16
  // rows, whole words, but for the last.
  uint32_t left = steps ? u1 - u0 : 0, ltile = u0 % tiles, lpass = u0 / tiles, ls = 0, lslot = 0, issued = 0;
  const uint8_t* lsc = nullptr;
  int lrest = 0, lx = 0, lrow = 0, lentry = 0;
  bool third = false;
  auto aim = [&]() {
    const uint64_t first = first_scale(lpass, ltile, lane >> 1), word = (first & ~3ull) + 4 * (lane & 1);
    lsc = a.scales + word;
    lrest = word < scale_bytes ? (int)min(scale_bytes - word, (uint64_t)0x40000000u) : 0;
    third = !(lane & 1) && (first & 3);
    lrow = (int)first_row(ltile);
    lentry = (int)passes[lpass].e;
  };
  const uint32_t scale_to = scale_ring + (lane >> 1) * kScaleWords * 4 + (lane & 1) * 4;
  auto load = [&]() {
    if (left) {
      if (lane == 0) {
        const uint32_t bar = smem_u32(&landed[warp][lslot]);
        mbar_expect_tx(bar, kCodeBytes);
        tma_load_3d(ring + lslot * kCodeBytes, &tw, lx, lrow, lentry, bar);
      }
      if (lrest > 0) copy4(scale_to + lslot * kScaleBytes, lsc, (uint32_t)min(4, lrest));
      if (third && lrest > 8) copy4(scale_to + lslot * kScaleBytes + 8, lsc + 8, (uint32_t)min(4, lrest - 8));
      lsc += kStageBlocks, lrest -= kStageBlocks, lx += kStageBlocks * 16;
      ++issued;
      if (++ls == steps) {
        ls = 0, --left;
        lx = (int)(s0 * kStageBlocks * 16);
        if (++ltile == tiles) ltile = 0, ++lpass;
        if (ltile != 0 && ltile + 1 != tiles) {
          lsc += kTileRows * blocks - steps * kStageBlocks;
          lrest -= (int)min(kTileRows * blocks - steps * kStageBlocks, (uint32_t)max(lrest, 0));
          lrow += kTileRows;
        } else if (left) {
          aim();
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    lslot = lslot + 1 == stages ? 0 : lslot + 1;
  };
  lx = (int)(s0 * kStageBlocks * 16);
  if (left) aim();
  __syncthreads();  // the barriers are ready
  for (uint32_t i = 0; i < stages - 1; ++i) load();

  uint32_t slot = 0, phase = 0, held = 0, shift = 0, tile = u0 % tiles, pass = u0 / tiles;
  bool lost = false;
  // The lane's blocks of a row's last stage, whose other scales are not the row's.
  const uint32_t ragged = blocks % kStageBlocks;
  const uint32_t ends = ragged - min(ragged, 4 * (lane & 1)), keep = ends < 4 ? (1u << 8 * ends) - 1 : 0xffffffffu;
  // Columns without a row take another's (R < 4) or what is there: each
  // column is its own, and theirs are not stored.
  const uint4* const x0 = reinterpret_cast<const uint4*>(xs) + (((g >> 1) % R) * 4 + t) * 2 + (g & 1);
  const float* const sx0 = sxs + t % R;
  uint32_t large = 0;  // bits 6 and 7 of a scale byte, of the held units' bytes: those of kLarge
  auto group_sync = [&]() {
    if (share > 1)
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * share) : "memory");
    else
      __syncwarp();
  };
  for (uint32_t u = u0; u < u1; ++u, ++tile) {
    if (tile == tiles) tile = 0, ++pass;
    const Pass ps = passes[pass];
    if (tile == 0 || u == u0) {
      // The warp's part of the pass's inputs: a row and stage at a time, 8
      // inputs a lane; zeros past the row's end.
      __syncwarp();
      for (uint32_t r = 0; r < ps.count; ++r) {
        const uint32_t p = perm[ps.first + r];
        const typename E::Storage* x = static_cast<const typename E::Storage*>(a.x) + (size_t)(p & 0xFFFFu) * a.ldx +
                                       (a.per_rank ? (size_t)(p >> 16) * a.kk : 0);
        const bool wide = ((uintptr_t)x & 15) == 0;
#pragma unroll 2
        for (uint32_t step = 0; step < steps; ++step) {
          const uint32_t c = step * kStageBlocks + (lane >> 2), q = lane & 3;
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = 0.0f;
          if (s0 * kStageBlocks + c < blocks) mx::load8<E>(x, 32 * (s0 * kStageBlocks + c) + 8 * q, wide, v);
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) top = max(top, mx::finite_bits(v[j]));
          const int up = mx::input_shift<E>(__reduce_max_sync(0xffffffffu, top));
          uint32_t hi[4], lo[4];
          mx::split8<true>(v, mx::scale_value((uint32_t)(127 + up)), hi, lo);
          uint4* to = reinterpret_cast<uint4*>(xs) + ((c * R + r) * 4 + q) * 2;
          to[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          to[1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          if (lane == 0) sxs[step * R + r] = mx::power_of_two(-up - kMoved);
        }
      }
      __syncwarp();
    }
    // Where the scale bytes of row lane / 2 lie in their words (a stage moves on by whole words).
    if (tile == 0 || tile + 1 == tiles || u == u0) shift = 8 * ((uint32_t)first_scale(pass, tile, lane >> 1) & 3u);
    float acc0 = 0.0f, acc1 = 0.0f;
    const uint4* xat = x0;
    const float* sat = sx0;
    for (uint32_t step = 0; step < steps; ++step) {
      load();
      asm volatile("cp.async.wait_group %0;" ::"n"(stages - 1) : "memory");  // all but the last ones
      const uint32_t bar = smem_u32(&landed[warp][slot]);
      if (!mbar_try(bar, phase) && !lost && !mbar_wait(bar, phase, wait_cycles)) {
        lost = true;  // the results are not to be used: the status says so
        record(err, LS_TIMEOUT);
      }
      __syncwarp();
      // The stage's scales as factors, four blocks of one row a lane: 2^(byte -
      // 127 + kMoved), so that a byte is its factor's exponent. Blocks past
      // the row's end have zeros for codes and inputs, and any factor.
      {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(mine_smem + slot * kScaleBytes) +
                            (lane >> 1) * kScaleWords + (lane & 1);
        uint32_t bytes = __funnelshift_r(w[0], w[1], shift), f[4];
        if (ragged && s0 + step + 1 == all_steps) bytes &= keep;
        large |= bytes & (bytes << 1);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          f[j] = ((j < 3 ? bytes << (23 - 8 * j) : bytes >> 1) & 0x7F800000u) + ((uint32_t)kMoved << 23);
        reinterpret_cast<uint4*>(factors)[lane] = make_uint4(f[0], f[1], f[2], f[3]);
      }
      __syncwarp();
      const uint8_t* st = smem + (warp * stages + slot) * kCodeBytes + g * 128 + t * 4;
      const float4* fg = reinterpret_cast<const float4*>(factors) + 2 * g;
      float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
      for (uint32_t b4 = 0; b4 < kStageBlocks; b4 += 4) {
        const float4 f0 = fg[b4 / 4], f1 = fg[16 + b4 / 4];
        const float s0v[4] = {f0.x, f0.y, f0.z, f0.w}, s1v[4] = {f1.x, f1.y, f1.z, f1.w};
#pragma unroll
        for (uint32_t bb = 0; bb < 4; ++bb) {
          const uint32_t b = b4 + bb;
          const uint8_t* at = st + ((b ^ g) << 4);  // the 128-byte swizzle
          float v0, v1;  // the block's sums, times its factors
          block_sums(*reinterpret_cast<const uint32_t*>(at), *reinterpret_cast<const uint32_t*>(at + 8 * 128),
                     xat[b * R * 8], v0, v1);
          sum0 = fmaf(v0, s0v[bb], sum0);
          sum1 = fmaf(v1, s1v[bb], sum1);
        }
      }
      const float sx = *sat;
      acc0 = fmaf(sum0, sx, acc0);
      acc1 = fmaf(sum1, sx, acc1);
      xat += kStageBlocks * R * 8, sat += R;
      if (++slot == stages) slot = 0, phase ^= 1;
      __syncwarp();  // before the stage is loaded again
    }
    // The warps' sums of up to `batch` units of a pass are added together at
    // once: a barrier a unit, and the adding behind it, held the warps up for
    // as long as half a unit's products.
    float(*rd)[kTileRows * R] = red[held];
    if (t < (uint32_t)R) {
      rd[warp][t * kTileRows + g] = acc0;
      rd[warp][t * kTileRows + g + 8] = acc1;
    }
    if (++held < batch && u + 1 < u1 && tile + 1 < tiles) continue;
    // Their rows with large scales are summed again first, while the pass's inputs
    // are here. (One look for all of them: a vote and a branch a stage cost 3%, one
    // place of it: a second one, or a call, 2%.)
    if (__any_sync(0xffffffffu, large & 0x80808080u)) {
#pragma unroll 1
      for (uint32_t h = 0; h < held; ++h) {
        const uint64_t row = (uint64_t)passes[pass].e * a.n + first_row(tile + 1 - held + h) + g;
        sum_large(a.w + row * (a.kk / 2) + 4 * t, a.scales + row * blocks, blocks, s0 * kStageBlocks,
                  min((s0 + steps) * kStageBlocks, blocks), x0, sx0, R, t < (uint32_t)R,
                  &red[h][warp][t * kTileRows + g]);
      }
      large = 0;
    }
    group_sync();
    for (uint32_t o = part * 32 + lane; o < held * (kTileRows * R); o += 32 * share) {
      const uint32_t uo = u + 1 - held + o / (kTileRows * R), i = o % (kTileRows * R);
      const Pass po = passes[uo / tiles];
      if ((i >> 4) >= po.count) continue;
      const float* from = &red[o / (kTileRows * R)][group * share][i];
      float v = from[0];
#pragma unroll 4
      for (uint32_t w = 1; w < share; ++w) v = __fadd_rn(v, from[w * (kTileRows * R)]);
      const uint32_t p = perm[po.first + (i >> 4)];
      mx::store<E>(static_cast<typename E::Storage*>(a.y) + (size_t)(p & 0xFFFFu) * a.ldy + (size_t)(p >> 16) * a.n +
                       first_row(uo % tiles) + (i & 15),
                   v);
    }
    held = 0;
    group_sync();
  }
  // Every stage issued was waited for above, so none is in flight (unless
  // one was lost: then what is still out is waited for here, within limits).
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (lost)
    for (uint32_t i = issued > stages ? issued - stages : 0; i < issued; ++i)
      mbar_wait(smem_u32(&landed[warp][i % stages]), (i / stages) & 1, wait_cycles);
}

// How many warps share a unit: the fewest rounds of units, each its blocks
// a warp and about 8 blocks' worth of fixed cost, and the inputs' splitting
// before them, whose inputs fit (4096 x 11008 by one row: 16 warps 11.4 us, 8
// 12.9). Each group of warps has its own copy of the inputs, so at 4 rows a pass
// it is often shared memory that decides: K = 1408 leaves 8 warps a unit, where
// the costs alone would take 2. 0: none.
inline uint32_t share_of(uint64_t units, uint32_t blocks, uint32_t R, int sms) {
  uint32_t best = 0;
  uint64_t least = ~0ull;
  const uint32_t all = (blocks + kStageBlocks - 1) / kStageBlocks;
  for (uint32_t share = kWarps; share >= 1; share /= 2) {
    const uint32_t steps = (all + share - 1) / share;
    const uint64_t at_once = (uint64_t)sms * (kWarps / share);
    const uint64_t cost = (units + at_once - 1) / at_once * (steps * kStageBlocks + 8) + 4 * steps;
    if (kStaticBytes + block_bytes(all, share, kLeastBatch, R) <= kSmemBudget && cost < least)
      least = cost, best = share;
  }
  return best;
}

// [entries][n][kk / 2] bytes of codes as boxes of 128 bytes x 16 rows,
// 128-byte swizzle; zeros past a row's end.
inline bool code_map(CUtensorMap* map, const FkLinearMx& a) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return false;
    fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  cuuint64_t dims[3] = {a.kk / 2, a.n, a.entries};
  cuuint64_t strides[2] = {a.kk / 2, (cuuint64_t)a.kk / 2 * a.n};
  cuuint32_t box[3] = {128, kTileRows, 1}, estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(a.w), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class E, int R>
cudaError_t launch(const FkLinearMx& a, uint32_t share, int sms, int* err, bool pdl, cudaStream_t s) {
  const uint64_t pairs = (uint64_t)a.m * a.k, tiles = (a.n + kTileRows - 1) / kTileRows;
  const uint32_t all = (a.kk / mx::kBlock + kStageBlocks - 1) / kStageBlocks;
  const uint32_t batch = kStaticBytes + block_bytes(all, share, kBatch, R) <= kSmemBudget ? kBatch : kLeastBatch;
  size_t rest = block_bytes(all, share, batch, R) - (size_t)kWarps * kStages * kCodeBytes;
  if (a.ids && rest < (a.entries + kThreads) * 4) rest = (a.entries + kThreads) * 4;  // the count's space
  const size_t smem = 1024 + (size_t)kWarps * kStages * kCodeBytes + rest;
  CUtensorMap tw;
  if (!code_map(&tw, a)) return cudaErrorInvalidValue;
  cudaError_t e = fk_allow_smem(stream_kernel<E, R>, smem);
  if (e != cudaSuccess) return e;
  const uint64_t most = (pairs * tiles + kWarps / share - 1) / (kWarps / share);  // blocks that have a unit
  return fk_launch_ex(stream_kernel<E, R>, dim3((uint32_t)(most < (uint64_t)sms ? most : (uint64_t)sms)),
                      dim3(kThreads), smem, s, pdl, tw, a, share, batch, (long long)4000000000LL, err);
}

}  // namespace ls
}  // namespace fk

size_t fk_linear_mxfp4_work(uint64_t entries, uint64_t n, uint64_t kk, uint64_t m, uint64_t k) {
  const uint64_t pairs = m * k;
  return 5 * pairs * kk + 16 * (pairs < 512 ? pairs : 512) * n + 16 * pairs + 64 * entries + 65536;
}

// Weights read again rather than widened by the tile kernel, whose launches
// and first loads cost as much as these (8 rows, two passes, by 4096 x 4096:
// 11.4 us, 19.2 in tiles; by 11008 x 4096 19.5 and 21.1, by 32000 x 4096 44.1
// and 30.0; 16 rows by 2048 x 2048 8.3 and 12.7, 64 by 1024 x 2048 12.3 and 13.0).
constexpr uint64_t kAgain = 64u << 20;

// The rows a pass of the streaming kernel and the warps a unit for a call; warps
// 0: the call goes to tiles.
struct FkStream {
  uint32_t R, share;
};
static FkStream stream_of(const FkLinearMx& a, int sms) {
  const uint64_t pairs = (uint64_t)a.m * a.k;
  const uint64_t experts = a.ids && pairs > a.entries ? a.entries : a.ids ? pairs : 1;  // at most
  // A pass over an expert's weights for every 4 of its pairs.
  const uint64_t passes = (pairs + 4 * experts - 1) / (4 * experts);
  // Routed tiles gain past two (16 experts of 512 x 512, 64 rows' 4 each: 15.3
  // us in passes, 13.4 in tiles) and over a quarter of the weights (64 experts
  // of 1024 x 1024, 128 rows' 4 each: 38 us in two, 31 in tiles), dense ones
  // past 16 (500 rows by 1024 x 128: 13.3 us in passes, 8.5 in tiles).
  if (pairs > fk::ls::kMaxPairs || a.n < fk::ls::kTileRows || passes > (a.ids ? 2 : 16) ||
      (passes - 1) * experts * a.n * a.kk > (a.ids ? kAgain / 4 : kAgain))
    return {0, 0};
  // Rows a pass: 4, fewer where there are no more or where they do not fit.
  for (uint32_t R = pairs <= 2 ? (uint32_t)pairs : 4; R >= 1; R /= 2) {
    const uint64_t units = experts * ((pairs + R * experts - 1) / (R * experts)) *
                           ((a.n + fk::ls::kTileRows - 1) / fk::ls::kTileRows);
    if (const uint32_t share = fk::ls::share_of(units, a.kk / 32, R, sms)) return {R, share};
  }
  return {0, 0};
}

uint32_t fk_linear_mxfp4_tokens(const FkLinearMx& a, FkElem e, int sms) {
  return stream_of(a, sms).share ? 0 : fk_linear_mxfp4_tile_tokens(a, e, sms);
}

cudaError_t fk_launch_linear_mxfp4(const FkLinearMx& a, FkElem e, int sms, int* err, bool pdl, cudaStream_t s) {
  if (a.m == 0 || a.n == 0) return cudaSuccess;
  if (a.kk == 0 || a.kk % fk::mx::kBlock != 0 || a.k == 0 || a.entries == 0 || a.entries > fk::ls::kMaxEntries ||
      a.ldx < (uint64_t)a.kk * (a.per_rank ? a.k : 1) || a.ldy < (uint64_t)a.k * a.n)
    return cudaErrorInvalidValue;
  const FkStream v = stream_of(a, sms);
  if (!v.share) return fk_launch_linear_mxfp4_tile(a, e, sms, err, pdl, s);
#define FK_CALL(E)                                                  \
  (v.R == 1   ? fk::ls::launch<E, 1>(a, v.share, sms, err, pdl, s)   \
   : v.R == 2 ? fk::ls::launch<E, 2>(a, v.share, sms, err, pdl, s)   \
              : fk::ls::launch<E, 4>(a, v.share, sms, err, pdl, s))
  return FK_BY_ELEM(e, FK_CALL);
#undef FK_CALL
}
