// Rows to microscaled 4-bit floating point and back (fk_mxfp4.cuh has the
// format). A block of 32 elements takes the scale 2^(floor(log2 amax) - 2),
// at least 2^-127, so that its largest magnitude lies in [4, 8) of it; the
// elements are rounded to nearest, ties to even, and past 6 to 6. A block
// with an infinity or a NaN takes the NaN scale (byte 255) and codes 0: all
// of its values are NaN.
//
// Both directions move their bytes once and are HBM's: 22016 x 4096 bf16 to
// codes and back 114 us together, 5.6 TB/s, 87% of what a copy reaches.
#include "fk_common.cuh"
#include "fk_kernels.h"
#include "fk_mxfp4.cuh"

namespace fk {
namespace mx {

// Groups of a thread in flight: as many bytes as HBM's latency asks for.
constexpr uint32_t kAhead = 4;

// Where group `at` of the rows (`size` elements, `groups` a row) is in an
// array whose rows are ld apart: rows back to back need no division, and few
// groups a 32-bit one.
__device__ __forceinline__ uint64_t place_of(uint64_t at, uint32_t size, uint32_t groups, uint32_t ld, bool few) {
  if (ld == size * groups) return size * at;
  const uint64_t r = few ? (uint32_t)at / groups : at / groups;
  return r * ld + size * (at - r * groups);
}

// A thread eight elements at a time, four threads a block of 32: the block's largest
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
  const uint64_t total = rows * eighths, stride = (uint64_t)gridDim.x * blockDim.x;
  const bool few = total < 0xFFFFFFFFull;
  const bool aligned = (uint64_t)ldx * sizeof(typename E::Storage) % 16 == 0;
  auto narrow = [&](uint64_t at, const float(&v)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    // The four threads of a block are in one warp and come here together.
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
    if ((at & 3u) == 0) scales[at >> 2] = (uint8_t)s;
  };
  uint64_t at = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x;
  if (aligned) {
    // The loads as they are, widened when their turn comes: 128 bytes of a
    // thread in flight in either width.
    constexpr uint32_t kVecs = E::kElem == FK_F32 ? 2 : 1, kDeep = 8 / kVecs;
    for (; at + (kDeep - 1) * stride < total; at += kDeep * stride) {
      uint4 raw[kDeep][kVecs];
#pragma unroll
      for (uint32_t u = 0; u < kDeep; ++u)
#pragma unroll
        for (uint32_t h = 0; h < kVecs; ++h)
          raw[u][h] = __ldg(reinterpret_cast<const uint4*>(x + place_of(at + u * stride, 8, eighths, ldx, few)) + h);
#pragma unroll
      for (uint32_t u = 0; u < kDeep; ++u) {
        float v[8];
        if constexpr (E::kElem == FK_F32) {
          const uint32_t w[8] = {raw[u][0].x, raw[u][0].y, raw[u][0].z, raw[u][0].w,
                                 raw[u][kVecs - 1].x, raw[u][kVecs - 1].y, raw[u][kVecs - 1].z, raw[u][kVecs - 1].w};
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
        } else {
          const float4 a = E::widen4(make_uint2(raw[u][0].x, raw[u][0].y)),
                       b = E::widen4(make_uint2(raw[u][0].z, raw[u][0].w));
          v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
        narrow(at + u * stride, v);
      }
    }
  }
  for (; at < total; at += stride) {
    float v[8];
    load8<E>(x + place_of(at, 8, eighths, ldx, few), 0, aligned, v);
    narrow(at, v);
  }
}

// A thread four codes at a time, so that a warp's stores of f32 are whole
// lines (eight a thread, in two stores, left half of each sector to the other).
template <class E>
__global__ void __launch_bounds__(256) widen_kernel(const uint32_t* __restrict__ codes,
                                                    const uint8_t* __restrict__ scales, uint64_t rows, uint32_t k,
                                                    uint32_t ldy, typename E::Storage* __restrict__ y) {
  grid_wait();
  grid_launch_dependents();
  const uint32_t quarters = k / 4;
  const uint64_t total = rows * quarters, stride = (uint64_t)gridDim.x * blockDim.x;
  const bool aligned = (uint64_t)ldy * sizeof(typename E::Storage) % 16 == 0, few = total < 0xFFFFFFFFull;
  auto put = [&](uint64_t at, uint32_t w, uint32_t s) {
    uint32_t d[4];  // of the word's eight, this thread's four
    widen8_f16(w, d);
    const float f = scale_value(s);
    const float2 a = F16::widen2(at & 1 ? d[2] : d[0]), b = F16::widen2(at & 1 ? d[3] : d[1]);
    const float v[4] = {__fmul_rn(a.x, f), __fmul_rn(a.y, f), __fmul_rn(b.x, f), __fmul_rn(b.y, f)};
    typename E::Storage* to = y + place_of(at, 4, quarters, ldy, few);
    if (!aligned) {
#pragma unroll
      for (int j = 0; j < 4; ++j) store<E>(to + j, v[j]);
    } else if constexpr (E::kElem == FK_F32) {
      *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      typename E::Storage h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) store<E>(h + j, v[j]);
      *reinterpret_cast<uint2*>(to) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    }
  };
  uint64_t at = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x;
  for (; at + (kAhead - 1) * stride < total; at += kAhead * stride) {
    uint32_t w[kAhead], s[kAhead];
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      w[u] = __ldg(codes + ((at + u * stride) >> 1));
      s[u] = __ldg(scales + ((at + u * stride) >> 3));
    }
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) put(at + u * stride, w[u], s[u]);
  }
  for (; at < total; at += stride) put(at, __ldg(codes + (at >> 1)), __ldg(scales + (at >> 3)));
}

// `a_sm` blocks an SM at most: 4 of the quantisation (1024 threads, 128 bytes
// of each in flight), 64 of the widening, whose stores run out
// better in short blocks (22016 x 4096: 66 us, 81 us with 8).
static unsigned grid_for(uint64_t threads, uint64_t a_sm) {
  const uint64_t b = (threads + 255) / 256;
  return (unsigned)(b > 148ull * a_sm ? 148ull * a_sm : b);
}

}  // namespace mx
}  // namespace fk

cudaError_t fk_launch_quant_mxfp4(const void* x, FkElem e, uint64_t rows, uint32_t k, uint32_t ldx, uint8_t* codes,
                                  uint8_t* scales, bool pdl, cudaStream_t s) {
  if (rows == 0 || k == 0) return cudaSuccess;
  if (k % fk::mx::kBlock != 0 || ldx < k) return cudaErrorInvalidValue;
#define FK_CALL(E)                                                                                                 \
  fk_launch_ex(fk::mx::quant_kernel<E>, dim3(fk::mx::grid_for(rows * (k / 8), 4)), dim3(256), 0, s, pdl,              \
               static_cast<const E::Storage*>(x), rows, k, ldx, reinterpret_cast<uint32_t*>(codes), scales)
  return FK_BY_ELEM(e, FK_CALL);
#undef FK_CALL
}

cudaError_t fk_launch_widen_mxfp4(const uint8_t* codes, const uint8_t* scales, uint64_t rows, uint32_t k,
                                  uint32_t ldy, void* y, FkElem e, bool pdl, cudaStream_t s) {
  if (rows == 0 || k == 0) return cudaSuccess;
  if (k % fk::mx::kBlock != 0 || ldy < k) return cudaErrorInvalidValue;
#define FK_CALL(E)                                                                                      \
  fk_launch_ex(fk::mx::widen_kernel<E>, dim3(fk::mx::grid_for(rows * (k / 4), 64)), dim3(256), 0, s, pdl,   \
               reinterpret_cast<const uint32_t*>(codes), scales, rows, k, ldy, static_cast<E::Storage*>(y))
  return FK_BY_ELEM(e, FK_CALL);
#undef FK_CALL
}
