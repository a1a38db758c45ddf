// Microscaled 4-bit floating point (MXFP4): 32 consecutive elements of a row
// share a power-of-two scale. An element is a 4-bit code: sign, two exponent
// bits, one mantissa bit; 0, .5, 1, 1.5, 2, 3, 4, 6 by magnitude. Two codes
// a byte, the even element in the low half. The scale is a byte s, 2^(s -
// 127); s = 255 makes the block NaN. A row of k elements is k / 2 bytes of
// codes and k / 32 bytes of scales, rows back to back.
//
// Every value is code x scale, exact in binary32 (and in bfloat16) but past
// the type's largest: 1 to 3 significant bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "fk_elem16.cuh"

namespace fk {
namespace mx {

constexpr uint32_t kBlock = 32;  // elements a scale

// Eight codes of a word, as four binary16 pairs in element order (exact).
__device__ __forceinline__ void widen8_f16(uint32_t w, uint32_t (&d)[4]) {
  asm("{\n\t.reg .b8 a, b, c, e;\n\t"
      "mov.b32 {a, b, c, e}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, e;\n\t}"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(w));
}

// A scale byte's value: 2^(s - 127), subnormal at s = 0, NaN at s = 255.
__device__ __forceinline__ float scale_value(uint32_t s) {
  return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7FC00000u : s << 23);
}

// 2^e, e in -149 .. 127, and the e of such a power.
__device__ __forceinline__ float power_of_two(int e) {
  return __uint_as_float(e >= -126 ? (uint32_t)(e + 127) << 23 : 1u << (e + 149));
}
__device__ __forceinline__ int exponent_of(float power) {
  const uint32_t b = __float_as_uint(power);
  return b >> 23 ? (int)(b >> 23) - 127 : -118 - __clz(b);
}

// v 2^e + sum, |v| < 2^100, e at most 254, in two steps to the same side: what
// leaves binary32's range on the way is out of it at the end.
__device__ __forceinline__ float add_scaled(float v, int e, float sum) {
  const int at = max(e, -252), half = at >> 1;  // (2^-252 already leaves nothing)
  return fmaf(__fmul_rn(v, __uint_as_float((uint32_t)(half + 127) << 23)),
              __uint_as_float((uint32_t)(at - half + 127) << 23), sum);
}

// Two elements to codes: to nearest, ties to even, past 6 to 6; `lo` in the
// low half of the byte.
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\t"
      "cvt.u32.u8 %0, t;\n\t}"
      : "=r"(r)
      : "f"(hi), "f"(lo));
  return r;
}

// Eight consecutive elements of a row from element i on (a multiple of 8),
// widened to binary32. `wide`: the row's address is 16-byte aligned.
template <class E>
__device__ __forceinline__ void load8(const typename E::Storage* p, uint32_t i, bool wide, float (&v)[8]) {
  if constexpr (E::kElem == FK_F32) {
    if (wide) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p + i));
      const float4 b = __ldg(reinterpret_cast<const float4*>(p + i) + 1);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __ldg(p + i + j);
    }
  } else {
    if (wide) {
      const uint4 r = __ldg(reinterpret_cast<const uint4*>(p + i));
      const float4 a = E::widen4(make_uint2(r.x, r.y)), b = E::widen4(make_uint2(r.z, r.w));
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = E::widen(__ldg(p + i + j));
    }
  }
}

// How far to move a run of inputs so that binary16 holds them best: the
// power of two that takes the largest finite magnitude (its bits) into
// [2^14, 2^15), at most 2^127. Binary16 inputs stay as they are.
template <class E>
__device__ __forceinline__ int input_shift(uint32_t top) {
  if (E::kElem == FK_F16 || top == 0) return 0;
  return min(141 - (int)(top >> 23), 127);
}

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}

// Eight inputs times `by` as binary16 pairs, and what those leave (exact in
// binary32; nothing of an infinity or a NaN) as binary16 pairs again.
template <bool LOW>
__device__ __forceinline__ void split8(const float (&v)[8], float by, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float s0 = __fmul_rn(v[2 * i], by), s1 = __fmul_rn(v[2 * i + 1], by);
    const __half h0 = __float2half_rn(s0), h1 = __float2half_rn(s1);
    hi[i] = (uint32_t)__half_as_ushort(h0) | (uint32_t)__half_as_ushort(h1) << 16;
    if constexpr (LOW) {
      const float l0 = isfinite(s0) ? __fsub_rn(s0, __half2float(h0)) : 0.0f;
      const float l1 = isfinite(s1) ? __fsub_rn(s1, __half2float(h1)) : 0.0f;
      lo[i] = (uint32_t)__half_as_ushort(__float2half_rn(l0)) | (uint32_t)__half_as_ushort(__float2half_rn(l1)) << 16;
    }
  }
}

// A binary32 result stored in the output's type: rounded once, to nearest.
template <class E>
__device__ __forceinline__ void store(typename E::Storage* p, float v) {
  if constexpr (E::kElem == FK_F32)
    *p = v;
  else if constexpr (E::kElem == FK_BF16)
    *p = __bfloat16_as_ushort(__float2bfloat16_rn(v));
  else
    *p = __half_as_ushort(__float2half_rn(v));
}

// The same where `on`, without a branch: many of them in a row keep going.
template <class E>
__device__ __forceinline__ void store_if(bool on, typename E::Storage* p, float v) {
  if constexpr (E::kElem == FK_F32) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t@q st.global.f32 [%1], %2;\n\t}" ::"r"((int)on),
                 "l"(p), "f"(v)
                 : "memory");
  } else {
    const uint16_t h = E::kElem == FK_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t@q st.global.u16 [%1], %2;\n\t}" ::"r"((int)on),
                 "l"(p), "h"(h)
                 : "memory");
  }
}

}  // namespace mx
}  // namespace fk

// The launch for any element type, CALL(tag).
#define FK_BY_ELEM(e, CALL) \
  ((e) == FK_F32 ? CALL(fk::F32) : (e) == FK_BF16 ? CALL(fk::Bf16) : (e) == FK_F16 ? CALL(fk::F16) : cudaErrorInvalidValue)
