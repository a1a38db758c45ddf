// Rows to microscaled 4-bit floating point and back (fk_mxfp4.cuh has the
// format). A block of 32 elements takes the scale 2^(floor(log2 amax) - 2),
// at least 2^-127, so that its largest magnitude lies in [4, 8) of it; the
// elements are rounded to nearest, ties to even, and past 6 to 6. A block
// with an infinity or a NaN takes the NaN scale (byte 255) and codes 0: all
// of its values are NaN.
#include "fk_common.cuh"
#include "fk_kernels.h"
#include "fk_mxfp4.cuh"

namespace fk {
namespace mx {

// A thread eight elements, four threads a block of 32: the block's largest
// magnitude through two exchanges of bit patterns (which order as the
// magnitudes do, infinities and NaNs above), then four bytes of codes a
// thread.
template <class E>
__global__ void __launch_bounds__(256) quant_kernel(const typename E::Storage* __restrict__ x, uint64_t rows,
                                                    uint32_t k, uint32_t ldx, uint32_t* __restrict__ codes,
                                                    uint8_t* __restrict__ scales) {
  grid_wait();
  grid_launch_dependents();
  const uint32_t eighths = k / 8;
  const uint64_t total = rows * eighths;
  const bool aligned = (uint64_t)ldx * sizeof(typename E::Storage) % 16 == 0;
  for (uint64_t at = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x; at < total;
       at += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t r = at / eighths;
    const uint32_t c = (uint32_t)(at - r * eighths);
    float v[8];
    load8<E>(x + r * ldx, 8 * c, aligned, v);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    // The four threads of a block are in one warp and leave the loop together.
    const uint32_t quad = 0xFu << (threadIdx.x & 28u);
    top = max(top, __shfl_xor_sync(quad, top, 1));
    top = max(top, __shfl_xor_sync(quad, top, 2));
    const uint32_t e = top >> 23;
    const bool odd = e == 255;
    const uint32_t s = odd ? 255u : e > 2 ? e - 2 : 0u;
    const float by = __uint_as_float(odd ? 0u : (254u - s) << 23);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w |= narrow2(__fmul_rn(v[2 * j], by), __fmul_rn(v[2 * j + 1], by)) << (8 * j);
    codes[at] = odd ? 0u : w;
    if ((c & 3u) == 0) scales[at >> 2] = (uint8_t)s;
  }
}

// A thread eight codes.
template <class E>
__global__ void __launch_bounds__(256) widen_kernel(const uint32_t* __restrict__ codes,
                                                    const uint8_t* __restrict__ scales, uint64_t rows, uint32_t k,
                                                    uint32_t ldy, typename E::Storage* __restrict__ y) {
  grid_wait();
  grid_launch_dependents();
  const uint32_t eighths = k / 8;
  const uint64_t total = rows * eighths;
  const bool aligned = (uint64_t)ldy * sizeof(typename E::Storage) % 16 == 0;
  for (uint64_t at = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x; at < total;
       at += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t r = at / eighths;
    const uint32_t c = (uint32_t)(at - r * eighths);
    float v[8];
    widen8(__ldg(codes + at), v);
    const float s = scale_value(__ldg(scales + (at >> 2)));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], s);
    typename E::Storage* to = y + r * ldy + 8 * c;
    if (!aligned) {
#pragma unroll
      for (int j = 0; j < 8; ++j) store<E>(to + j, v[j]);
    } else if constexpr (E::kElem == FK_F32) {
      reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = (uint32_t)E::narrow(v[2 * j]) | (uint32_t)E::narrow(v[2 * j + 1]) << 16;
      *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
}

static unsigned grid_for(uint64_t threads) {
  const uint64_t b = (threads + 255) / 256;
  return (unsigned)(b > 148ull * 64 ? 148ull * 64 : b);
}

}  // namespace mx
}  // namespace fk

cudaError_t fk_launch_quant_mxfp4(const void* x, FkElem e, uint64_t rows, uint32_t k, uint32_t ldx, uint8_t* codes,
                                  uint8_t* scales, bool pdl, cudaStream_t s) {
  if (rows == 0 || k == 0) return cudaSuccess;
  if (k % fk::mx::kBlock != 0 || ldx < k) return cudaErrorInvalidValue;
#define FK_CALL(E)                                                                                                 \
  fk_launch_ex(fk::mx::quant_kernel<E>, dim3(fk::mx::grid_for(rows * (k / 8))), dim3(256), 0, s, pdl,              \
               static_cast<const E::Storage*>(x), rows, k, ldx, reinterpret_cast<uint32_t*>(codes), scales)
  return FK_BY_ELEM(e, FK_CALL);
#undef FK_CALL
}

cudaError_t fk_launch_widen_mxfp4(const uint8_t* codes, const uint8_t* scales, uint64_t rows, uint32_t k,
                                  uint32_t ldy, void* y, FkElem e, bool pdl, cudaStream_t s) {
  if (rows == 0 || k == 0) return cudaSuccess;
  if (k % fk::mx::kBlock != 0 || ldy < k) return cudaErrorInvalidValue;
#define FK_CALL(E)                                                                                      \
  fk_launch_ex(fk::mx::widen_kernel<E>, dim3(fk::mx::grid_for(rows * (k / 8))), dim3(256), 0, s, pdl,   \
               reinterpret_cast<const uint32_t*>(codes), scales, rows, k, ldy, static_cast<E::Storage*>(y))
  return FK_BY_ELEM(e, FK_CALL);
#undef FK_CALL
}
