// Products with MXFP4 weights (fk_mxfp4.cuh): y[r, j] = W[ids[r, j]] x[r],
// or x[r, j] where each rank has its own input; a dense product is one
// expert that every row takes. x and y in f32, bf16 or f16; the products
// and sums in binary32, the result rounded once.
#include "fk_common.cuh"
#include "fk_kernels.h"
#include "fk_mxfp4.cuh"

namespace fk {
namespace lx {

constexpr int kPairsAPass = 8;
constexpr uint32_t kPairWindow = 1024;  // (row, rank) pairs a block lists at a time

// The plain kernel: a block a (expert, 8 output rows), a warp a row. It
// lists the (row, rank) pairs that chose its expert and takes up to 8 at a
// time: a lane a block of 32 weights, its dot with each pair's inputs, then
// the warp's sum.
template <class E>
__global__ void __launch_bounds__(256) plain_kernel(FkLinearMx a) {
  __shared__ uint32_t pairs[kPairWindow];
  __shared__ uint32_t npairs;
  const uint32_t e = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_wait();
  grid_launch_dependents();
  const uint32_t all = a.m * a.k;
  const uint32_t o = blockIdx.x * 8u + (uint32_t)warp;
  const uint32_t blocks = a.kk / mx::kBlock;
  const size_t row = (size_t)e * a.n + (o < a.n ? o : 0);
  const uint4* wr = reinterpret_cast<const uint4*>(a.w) + row * blocks;
  const uint8_t* sr = a.scales + row * blocks;
  const bool wide = (uint64_t)a.ldx * sizeof(typename E::Storage) % 16 == 0;
  const typename E::Storage* x = static_cast<const typename E::Storage*>(a.x);
  typename E::Storage* y = static_cast<typename E::Storage*>(a.y);
  for (uint32_t w0 = 0; w0 < all; w0 += kPairWindow) {
    const uint32_t w1 = min(all, w0 + kPairWindow);
    __syncthreads();
    if (warp == 0) {
      uint32_t c = 0;
      for (uint32_t base = w0; base < w1; base += 32u) {
        const uint32_t p = base + (uint32_t)lane;
        const bool hit = p < w1 && (!a.ids || a.ids[p] == e);
        const uint32_t mask = __ballot_sync(0xffffffffu, hit);
        if (hit) pairs[c + __popc(mask & ((1u << lane) - 1u))] = p;
        c += __popc(mask);
        // A pair without an expert: its segment is 0, written by expert 0's blocks.
        if (a.ids && e == 0 && p < w1 && a.ids[p] >= a.entries)
          for (uint32_t q = blockIdx.x * 8u; q < min(a.n, blockIdx.x * 8u + 8u); ++q)
            mx::store<E>(y + (size_t)(p / a.k) * a.ldy + (size_t)(p % a.k) * a.n + q, 0.0f);
      }
      if (lane == 0) npairs = c;
    }
    __syncthreads();
    const uint32_t P = npairs;
    if (P == 0 || o >= a.n) continue;
    for (uint32_t p0 = 0; p0 < P; p0 += kPairsAPass) {
      const uint32_t np = min((uint32_t)kPairsAPass, P - p0);
      float acc[kPairsAPass];
#pragma unroll
      for (int q = 0; q < kPairsAPass; ++q) acc[q] = 0.0f;
      for (uint32_t b = lane; b < blocks; b += 32) {
        const uint4 cw = __ldg(wr + b);
        const float s = mx::scale_value(__ldg(sr + b));
        const uint32_t words[4] = {cw.x, cw.y, cw.z, cw.w};
        float dot[kPairsAPass];
#pragma unroll
        for (int q = 0; q < kPairsAPass; ++q) dot[q] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float wv[8];
          mx::widen8(words[i], wv);
#pragma unroll
          for (int q = 0; q < kPairsAPass; ++q) {
            if ((uint32_t)q >= np) continue;
            const uint32_t pr = pairs[p0 + q], r = pr / a.k, j = pr % a.k;
            float xv[8];
            mx::load8<E>(x + (size_t)r * a.ldx + (a.per_rank ? (size_t)j * a.kk : 0), 32 * b + 8 * i, wide, xv);
#pragma unroll
            for (int t = 0; t < 8; ++t) dot[q] = fmaf(wv[t], xv[t], dot[q]);
          }
        }
#pragma unroll
        for (int q = 0; q < kPairsAPass; ++q) acc[q] = fmaf(dot[q], s, acc[q]);
      }
#pragma unroll
      for (int q = 0; q < kPairsAPass; ++q) {
        const float total = warp_sum(acc[q]);
        if ((uint32_t)q < np && lane == 0) {
          const uint32_t pr = pairs[p0 + q];
          mx::store<E>(y + (size_t)(pr / a.k) * a.ldy + (size_t)(pr % a.k) * a.n + o, total);
        }
      }
    }
  }
}

}  // namespace lx
}  // namespace fk

size_t fk_linear_mxfp4_work(uint64_t entries, uint64_t n, uint64_t kk, uint64_t m, uint64_t k) {
  const uint64_t pairs = m * k;
  return 5 * pairs * kk + 16 * (pairs < 512 ? pairs : 512) * n + 16 * pairs + 64 * entries + 65536;
}

cudaError_t fk_launch_linear_mxfp4(const FkLinearMx& a, FkElem e, int sms, int* err, bool pdl, cudaStream_t s) {
  if (a.m == 0 || a.n == 0) return cudaSuccess;
  if (a.kk == 0 || a.kk % fk::mx::kBlock != 0 || a.k == 0 || a.entries == 0 ||
      a.ldx < (uint64_t)a.kk * (a.per_rank ? a.k : 1) || a.ldy < (uint64_t)a.k * a.n)
    return cudaErrorInvalidValue;
  if ((uint64_t)a.m * a.k > 8ull * a.entries) return fk_launch_linear_mxfp4_tile(a, e, sms, err, pdl, s);
  const dim3 grid((a.n + 7) / 8, a.entries);
#define FK_CALL(E) fk_launch_ex(fk::lx::plain_kernel<E>, grid, dim3(256), 0, s, pdl, a)
  return FK_BY_ELEM(e, FK_CALL);
#undef FK_CALL
}
