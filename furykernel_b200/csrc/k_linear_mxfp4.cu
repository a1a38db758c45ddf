// Products with MXFP4 weights (fk_mxfp4.cuh): y[r, j] = W[ids[r, j]] x[r],
// or x[r, j] where each rank has its own input; a dense product is one
// expert that every row takes. x and y in f32, bf16 or f16; the products
// and sums in binary32, the result rounded once. Two kernels: the streaming
// one below for few rows an expert, the tcgen05 one
// (k_linear_mxfp4_tile.cu) for more.
//
// The streaming kernel reads every weight once for up to R rows and is held
// by HBM, so the arithmetic a weight has to be little: at 23 bytes (43
// weights) a cycle an SM there are three instructions a weight. The codes
// widen to binary16 two an instruction and go to the tensor cores' warp-wide
// products (16 weight rows x 16 of K x 8 columns) unscaled; a block of 32
// weights, two such products, is one scale, which multiplies the block's
// sums. The columns are the inputs: a row as two binary16 parts, x = h1 +
// h2 relative to the largest of a stage's 128 (within 2^-23 of x or 2^-39
// of that largest), so 8 columns are 4 rows. Sums of blocks are binary32.
#include "fk_common.cuh"
#include "fk_kernels.h"
#include "fk_mxfp4.cuh"

namespace fk {
namespace ls {

constexpr uint32_t kWarps = 16;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr uint32_t kTileRows = 16;     // weight rows of a unit
constexpr uint32_t kStageBlocks = 4;   // blocks of 32 weights a row a stage
constexpr uint32_t kStages = 4;        // a warp's own ring
constexpr uint32_t kPitch = 80;        // a row's 64 bytes of codes: rows 20 banks apart, no two of 8 alike
constexpr uint32_t kStageBytes = kTileRows * (kPitch + 8);
constexpr uint32_t kMaxPairs = 512;
constexpr uint32_t kMaxEntries = 4096;
constexpr uint32_t kInputBudget = 114 * 1024;  // the inputs of the warps' passes

// A warp's inputs: `blocks` blocks of R rows, 128 bytes each (two parts),
// and a factor a row and stage.
__host__ __device__ constexpr uint32_t input_bytes(uint32_t blocks, uint32_t R) {
  return blocks * R * 128 + ((blocks + kStageBlocks - 1) / kStageBlocks * R * 4 + 15) / 16 * 16;
}

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
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
__global__ void __launch_bounds__(kThreads, 1) stream_kernel(const FkLinearMx a, uint32_t share) {
  constexpr int NT = (R + 3) / 4;  // products of 8 columns
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Pass passes[kMaxPairs];
  __shared__ uint16_t perm[kMaxPairs];
  __shared__ uint32_t ids_s[kThreads];
  __shared__ float red[2][kWarps][kTileRows * R];
  __shared__ uint32_t sums[2][kWarps], npasses_s, nrest_s;
  uint8_t* rings = smem;                                        // [kWarps][kStages][kStageBytes]
  uint8_t* inputs = rings + kWarps * kStages * kStageBytes;     // [kWarps] input_bytes
  const uint32_t blocks = a.kk / mx::kBlock;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t pairs = a.m * a.k, tiles = (a.n + kTileRows - 1) / kTileRows;

  // The weights too may be the previous launch's (quant_mxfp4's): nothing is read before it is done.
  grid_wait();
  grid_launch_dependents();
  uint32_t npasses, rest = 0;
  if (a.ids) {
    // The pairs of each expert, in the input's space (not filled yet).
    uint32_t* count = reinterpret_cast<uint32_t*>(inputs);
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
    if (tid < pairs) perm[(own < a.entries ? count[own] : rest) + place] = (uint16_t)tid;
    __syncthreads();
    // Pairs without an expert: zeros.
    for (uint32_t q = rest + blockIdx.x; q < pairs; q += gridDim.x)
      for (uint32_t i = tid; i < a.n; i += kThreads)
        mx::store<E>(static_cast<typename E::Storage*>(a.y) + (size_t)(perm[q] / a.k) * a.ldy +
                         (size_t)(perm[q] % a.k) * a.n + i,
                     0.0f);
  } else {
    npasses = (pairs + R - 1) / R;
    if (tid < npasses) {
      passes[tid].first = (uint16_t)(tid * R);
      passes[tid].count = (uint16_t)min((uint32_t)R, pairs - tid * R);
      passes[tid].e = 0;
    }
    if (tid < pairs) perm[tid] = (uint16_t)tid;
    __syncthreads();
  }

  const uint32_t abreast = kWarps / share, group = warp / share, part = warp % share;
  const uint64_t units = (uint64_t)npasses * tiles, groups = (uint64_t)gridDim.x * abreast,
                 gid = (uint64_t)blockIdx.x * abreast + group;
  const uint32_t u0 = (uint32_t)(gid * units / groups), u1 = (uint32_t)((gid + 1) * units / groups);
  // This warp's blocks of every row.
  const uint32_t b0 = part * blocks / share, nb = (part + 1) * blocks / share - b0;
  const uint32_t steps = (nb + kStageBlocks - 1) / kStageBlocks;
  const uint32_t ring = smem_at(rings + warp * kStages * kStageBytes);
  const uint64_t scale_bytes = (uint64_t)a.entries * a.n * blocks;
  // The inputs, [blocks][R][4][2] 16 bytes as the products take them, and
  // the factors [steps][R].
  const uint32_t most_blocks = (blocks + share - 1) / share;
  uint8_t* xs = inputs + warp * input_bytes(most_blocks, R);
  float* sxs = reinterpret_cast<float*>(xs + most_blocks * R * 128);

  // The loads of the next stage: the warp's own cursor over (unit, step).
  // Addresses are formed once a unit and move on by a stage.
  uint32_t left = steps ? u1 - u0 : 0, ltile = u0 % tiles, lpass = u0 / tiles, ls = 0, lslot = 0;
  const uint8_t *lc0 = nullptr, *lc1 = nullptr, *lsc = nullptr;
  uint32_t loff = 0, lrest = 0;
  const uint32_t to0 = (lane >> 2) * kPitch + (lane & 3) * 16, to_scale = kTileRows * kPitch + lane * 4;
  auto load = [&]() {
    if (left) {
      if (ls == 0) {
        const uint64_t row0 = (uint64_t)passes[lpass].e * a.n;
        const uint32_t r0 = ltile * kTileRows;
        lc0 = a.w + ((row0 + min(r0 + (lane >> 2), a.n - 1)) * blocks + b0 + (lane & 3)) * 16;
        lc1 = a.w + ((row0 + min(r0 + (lane >> 2) + 8, a.n - 1)) * blocks + b0 + (lane & 3)) * 16;
        // A row's scales: the words that hold their bytes, wherever they
        // start; the table's last word may be short.
        const uint64_t first = (row0 + min(r0 + (lane >> 1), a.n - 1)) * blocks + b0;
        const uint64_t word = (first & ~3ull) + 4 * (lane & 1);
        loff = 4 * (lane & 1) - (uint32_t)(first & 3);  // where the word starts against the first byte
        lsc = a.scales + word;
        lrest = word < scale_bytes ? (uint32_t)min(scale_bytes - word, (uint64_t)0x40000000u) : 0u;
      }
      const uint32_t have = min(nb - ls * kStageBlocks, kStageBlocks), st = ring + lslot;
      if ((lane & 3) < have) {
        copy16(st + to0, lc0);
        copy16(st + to0 + 8 * kPitch, lc1);
      }
      if ((int)loff < (int)have) copy4(st + to_scale, lsc, min(4u, lrest));
      lc0 += kStageBlocks * 16, lc1 += kStageBlocks * 16, lsc += kStageBlocks, lrest -= kStageBlocks;
      if (++ls == steps) {
        ls = 0, --left;
        if (++ltile == tiles) ltile = 0, ++lpass;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    lslot = lslot == (kStages - 1) * kStageBytes ? 0 : lslot + kStageBytes;
  };
#pragma unroll
  for (uint32_t i = 0; i < kStages - 1; ++i) load();

  uint32_t slot = 0, tile = u0 % tiles, pass = u0 / tiles;
  for (uint32_t u = u0; u < u1; ++u, ++tile) {
    if (tile == tiles) tile = 0, ++pass;
    const Pass ps = passes[pass];
    if (tile == 0 || u == u0) {
      // The warp's part of the pass's inputs: 16 lanes a row and stage, 8
      // inputs a lane.
      __syncwarp();
      for (uint32_t i = lane >> 4; i < ps.count * steps; i += 2) {
        const uint32_t r = i / steps, step = i - r * steps, c = step * kStageBlocks + ((lane >> 2) & 3), q = lane & 3;
        const uint32_t p = perm[ps.first + r];
        const typename E::Storage* x = static_cast<const typename E::Storage*>(a.x) + (size_t)(p / a.k) * a.ldx +
                                       (a.per_rank ? (size_t)(p % a.k) * a.kk : 0);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        if (c < nb) mx::load8<E>(x, 32 * (b0 + c) + 8 * q, ((uintptr_t)x & 15) == 0, v);
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, mx::finite_bits(v[j]));
        const uint32_t mask = 0xFFFFu << (lane & 16u);  // the stage's lanes leave the loop together
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor_sync(mask, top, o));
        const int up = mx::input_shift<E>(top);
        uint32_t hi[4], lo[4];
        mx::split8<true>(v, mx::scale_value((uint32_t)(127 + up)), hi, lo);
        if (c < nb) {
          uint4* to = reinterpret_cast<uint4*>(xs) + ((c * R + r) * 4 + q) * 2;
          to[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          to[1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        if ((lane & 15) == 0) sxs[step * R + r] = mx::scale_value((uint32_t)(127 - up));
      }
      __syncwarp();
    }
    const uint64_t row0 = (uint64_t)ps.e * a.n;
    const uint32_t r0 = tile * kTileRows;
    float acc[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = 0.0f;
    // Where rows g and g + 8 have their scales' bytes in their words: a
    // stage moves on by whole words.
    uint32_t shift[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      shift[h] = 8 * ((uint32_t)((row0 + min(r0 + g + 8 * h, a.n - 1)) * blocks + b0) & 3u);
    // Columns without a row take another's (R < 4) or what is there: each
    // column is its own, and theirs are not stored.
    const uint4* xat = reinterpret_cast<const uint4*>(xs) + (((g >> 1) % R) * 4 + t) * 2 + (g & 1);
    const float* sat = sxs + t % R;
    for (uint32_t step = 0; step < steps; ++step) {
      load();
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      const uint8_t* st = rings + warp * kStages * kStageBytes + slot;
      slot = slot == (kStages - 1) * kStageBytes ? 0 : slot + kStageBytes;
      const uint32_t have = min(nb - step * kStageBlocks, kStageBlocks);
      uint32_t sc[2];  // four scale bytes of each row
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint2 w = *reinterpret_cast<const uint2*>(st + kTileRows * kPitch + (g + 8 * h) * 8);
        sc[h] = __funnelshift_r(w.x, w.y, shift[h]);
      }
      float sum[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) sum[j][0] = sum[j][1] = 0.0f;
      // One block of 32: two products, their sums times the block's scales.
      auto block = [&](uint32_t b, float s0, float s1) {
        uint32_t p[4], q[4];
        mx::widen8_f16(*reinterpret_cast<const uint32_t*>(st + g * kPitch + b * 16 + t * 4), p);
        mx::widen8_f16(*reinterpret_cast<const uint32_t*>(st + (g + 8) * kPitch + b * 16 + t * 4), q);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 x = xat[(b * R + 4 * j) * 8];
          float d[4];
          mma0(d, p[0], q[0], p[1], q[1], x.x, x.y);
          mma(d, p[2], q[2], p[3], q[3], x.z, x.w);
          sum[j][0] = fmaf(__fadd_rn(d[0], d[1]), s0, sum[j][0]);
          sum[j][1] = fmaf(__fadd_rn(d[2], d[3]), s1, sum[j][1]);
        }
      };
      // Scales of 2^-126 .. 2^127, nearly all: a byte is its factor's exponent.
      auto plain = [&](uint32_t b, uint32_t w) {
        return __uint_as_float((b < 3 ? w << (23 - 8 * b) : w >> 1) & 0x7F800000u);
      };
      const uint32_t odd = __vcmpeq4(sc[0], 0) | __vcmpeq4(sc[1], 0) | __vcmpeq4(sc[0], 0xFFFFFFFFu) |
                           __vcmpeq4(sc[1], 0xFFFFFFFFu);
      if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
        for (uint32_t b = 0; b < have; ++b)
          block(b, mx::scale_value((sc[0] >> (8 * b)) & 0xFFu), mx::scale_value((sc[1] >> (8 * b)) & 0xFFu));
      } else if (have == kStageBlocks) {
#pragma unroll
        for (uint32_t b = 0; b < kStageBlocks; ++b) block(b, plain(b, sc[0]), plain(b, sc[1]));
      } else {
#pragma unroll
        for (uint32_t b = 0; b < kStageBlocks - 1; ++b)
          if (b < have) block(b, plain(b, sc[0]), plain(b, sc[1]));
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float sx = sat[4 * j];
        acc[j][0] = fmaf(sum[j][0], sx, acc[j][0]);
        acc[j][1] = fmaf(sum[j][1], sx, acc[j][1]);
      }
      xat += kStageBlocks * R * 8, sat += R;
      __syncwarp();  // before the stage is loaded again
    }
    float(*rd)[kTileRows * R] = red[u & 1];
#pragma unroll
    for (int j = 0; j < NT; ++j)
      if (4 * j + t < (uint32_t)R) {
        rd[warp][(4 * j + t) * kTileRows + g] = acc[j][0];
        rd[warp][(4 * j + t) * kTileRows + g + 8] = acc[j][1];
      }
    if (share > 1)
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * share) : "memory");
    else
      __syncwarp();
    for (uint32_t i = part * 32 + lane; i < kTileRows * ps.count; i += 32 * share) {
      if (r0 + (i & 15) >= a.n) continue;
      float v = 0.0f;
      for (uint32_t w = 0; w < share; ++w) v = __fadd_rn(v, rd[group * share + w][i]);
      const uint32_t p = perm[ps.first + (i >> 4)];
      mx::store<E>(static_cast<typename E::Storage*>(a.y) + (size_t)(p / a.k) * a.ldy + (size_t)(p % a.k) * a.n + r0 +
                       (i & 15),
                   v);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// How many warps share a unit: the fewest rounds of units, each its blocks
// a warp and about 3 blocks' worth of fixed cost, and whose inputs fit.
inline uint32_t share_of(uint64_t units, uint32_t blocks, uint32_t R, int sms) {
  uint32_t best = 0;
  uint64_t least = ~0ull;
  for (uint32_t share = kWarps; share >= 1; share /= 2) {
    const uint32_t mine = (blocks + share - 1) / share;
    const uint64_t at_once = (uint64_t)sms * (kWarps / share), cost = (units + at_once - 1) / at_once * (mine + 3);
    if ((uint64_t)kWarps * input_bytes(mine, R) <= kInputBudget && cost < least) least = cost, best = share;
  }
  return best;
}

template <class E, int R>
cudaError_t launch(const FkLinearMx& a, uint32_t share, int sms, bool pdl, cudaStream_t s) {
  const uint64_t pairs = (uint64_t)a.m * a.k, tiles = (a.n + kTileRows - 1) / kTileRows;
  const uint32_t blocks = a.kk / mx::kBlock;
  size_t input = (size_t)kWarps * input_bytes((blocks + share - 1) / share, R);
  if (a.ids && input < (a.entries + kThreads) * 4) input = (a.entries + kThreads) * 4;  // the count's space
  const size_t smem = kWarps * kStages * kStageBytes + input;
  cudaError_t e = fk_allow_smem(stream_kernel<E, R>, smem);
  if (e != cudaSuccess) return e;
  const uint64_t most = (pairs * tiles + kWarps / share - 1) / (kWarps / share);  // blocks that have a unit
  return fk_launch_ex(stream_kernel<E, R>, dim3((uint32_t)(most < (uint64_t)sms ? most : (uint64_t)sms)),
                      dim3(kThreads), smem, s, pdl, a, share);
}

}  // namespace ls
}  // namespace fk

size_t fk_linear_mxfp4_work(uint64_t entries, uint64_t n, uint64_t kk, uint64_t m, uint64_t k) {
  const uint64_t pairs = m * k;
  return 5 * pairs * kk + 16 * (pairs < 512 ? pairs : 512) * n + 16 * pairs + 64 * entries + 65536;
}

cudaError_t fk_launch_linear_mxfp4(const FkLinearMx& a, FkElem e, int sms, int* err, bool pdl, cudaStream_t s) {
  if (a.m == 0 || a.n == 0) return cudaSuccess;
  if (a.kk == 0 || a.kk % fk::mx::kBlock != 0 || a.k == 0 || a.entries == 0 || a.entries > fk::ls::kMaxEntries ||
      a.ldx < (uint64_t)a.kk * (a.per_rank ? a.k : 1) || a.ldy < (uint64_t)a.k * a.n)
    return cudaErrorInvalidValue;
  const uint64_t pairs = (uint64_t)a.m * a.k;
  if (pairs <= fk::ls::kMaxPairs && pairs <= 8ull * a.entries) {
    // Rows a pass: 4 where an expert has that many on average, 8 past it,
    // fewer where there are no more or where they do not fit.
    uint32_t R = pairs <= 2 ? (uint32_t)pairs : pairs <= 4ull * a.entries ? 4 : 8, share = 0;
    const uint64_t experts = a.ids && pairs > a.entries ? a.entries : a.ids ? pairs : 1;  // at most
    for (; R >= 1; R /= 2) {
      const uint64_t passes = a.ids ? experts : (pairs + R - 1) / R;
      share = fk::ls::share_of(passes * ((a.n + fk::ls::kTileRows - 1) / fk::ls::kTileRows), a.kk / 32, R, sms);
      if (share) break;
    }
#define FK_CALL(E)                                          \
  (R == 1   ? fk::ls::launch<E, 1>(a, share, sms, pdl, s)   \
   : R == 2 ? fk::ls::launch<E, 2>(a, share, sms, pdl, s)   \
   : R == 4 ? fk::ls::launch<E, 4>(a, share, sms, pdl, s)   \
            : fk::ls::launch<E, 8>(a, share, sms, pdl, s))
    if (share) return FK_BY_ELEM(e, FK_CALL);
#undef FK_CALL
  }
  return fk_launch_linear_mxfp4_tile(a, e, sms, err, pdl, s);
}
