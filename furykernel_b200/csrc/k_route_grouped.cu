// The grouped router: a row's top k of n experts, for any number of rows.
//
//   s_i = sigmoid(x_i), 1 / (1 + exp(-x_i)), or softmax, exp(x_i - max) over
//         the row's sum of them;
//   c_i = s_i + bias_i (the balance bias; without one c_i = s_i);
//   a group (n / groups neighbouring experts) is worth the sum of its
//   group_by (1 or 2) largest c; the top_groups worthiest groups stay;
//   the k largest c of those groups are the row's experts, in that order;
//   w_j = s of expert j, over the k's sum in rank order when renorm, times
//   factor.
//
// Binary32 with one rounding an operation; each exponential, and a softmax
// row's sum of them, in binary64 rounded once, so that the scores, and with
// them the choice, do not depend on an order of addition. Ties go to the
// lower index; a NaN choice is below every number. A softmax row whose
// logits are all -inf has scores 0, and scores that sum to 0 give weights 0
// (a masked row: no NaN).
//
// A warp a row, its n / 32 scores a lane in registers as keys whose unsigned
// order is the choice's (NaN lowest), so that a round of the top k is two
// warp-wide reductions and no barrier. 8192 rows of 256 experts in 8 groups,
// top 8, sigmoid and bias: 20.5 us, 0.44 TB/s of the logits; the integer pipe
// bounds it (68% of its cycles: the rounds), not HBM (5%) nor the binary64
// exponentials.
#include "fk_common.cuh"
#include "fk_kernels.h"
#include "fk_mxfp4.cuh"

namespace fk {
namespace route {

constexpr uint32_t kAll = 0xffffffffu;

// Choices as keys that order as they do: 0 absent, 1 NaN, then the numbers.
__device__ __forceinline__ uint32_t key_of(float c) {
  if (isnan(c)) return 1u;
  const uint32_t b = __float_as_uint(c == 0.0f ? 0.0f : c);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  if (k <= 1u) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}

template <class E>
__device__ __forceinline__ float logit(const typename E::Storage* x, uint32_t i) {
  if constexpr (E::kElem == FK_F32)
    return __ldg(x + i);
  else
    return E::widen(__ldg(x + i));
}

// A warp a row, lane l holding experts l, l + 32, ...: T of them at most.
template <class E, int T>
__global__ void __launch_bounds__(128) route_grouped_kernel(FkRouteGrouped a) {
  grid_wait();
  grid_launch_dependents();
  const uint32_t lane = threadIdx.x & 31, r = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (r >= a.m) return;
  const typename E::Storage* x = static_cast<const typename E::Storage*>(a.x) + (size_t)r * a.ldx;
  float s[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const uint32_t i = lane + 32 * t;
    s[t] = i < a.n ? logit<E>(x, i) : -INFINITY;
  }
  if (a.sigmoid) {
#pragma unroll
    for (int t = 0; t < T; ++t) s[t] = __frcp_rn(__fadd_rn(1.0f, exp_rounded(-s[t])));
  } else {
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < T; ++t) top = max_number(top, s[t]);
    top = warp_max(top);
    double sum = 0.0;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      // Every logit -inf: 0 each, and a sum of 1.
      s[t] = lane + 32 * t >= a.n ? 0.0f : top == -INFINITY && !isnan(s[t]) ? 0.0f : exp_rounded(__fsub_rn(s[t], top));
      sum += (double)s[t];
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor_sync(kAll, sum, o);
    const float total = sum == 0.0 ? 1.0f : (float)sum;
#pragma unroll
    for (int t = 0; t < T; ++t) s[t] = __fdiv_rn(s[t], total);
  }
  uint32_t key[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const uint32_t i = lane + 32 * t;
    key[t] = i < a.n ? key_of(a.bias ? __fadd_rn(s[t], __ldg(a.bias + i)) : s[t]) : 0u;
  }
  if (a.top_groups < a.groups) {
    const uint32_t per = a.n / a.groups;
    uint32_t worth = 0;  // lane g: group g's worth
    // From each lane's largest two keys of group g.
    auto close = [&](uint32_t g, uint32_t k1, uint32_t k2) {
      uint32_t w = __reduce_max_sync(kAll, k1);
      if (a.group_by == 2 && per > 1) {
        // The largest but one: the first lane with the largest offers its second.
        const uint32_t has = __ballot_sync(kAll, k1 == w);
        const uint32_t m2 = __reduce_max_sync(kAll, lane == (uint32_t)__ffs(has) - 1 ? k2 : k1);
        w = key_of(__fadd_rn(of_key(w), of_key(m2)));
      }
      if (lane == g) worth = w;
    };
    uint32_t group[T];  // the group of each of the lane's experts
    if (per % 32 == 0) {  // a group is whole turns of the lanes: one pass
      uint32_t g = 0, left = per / 32, k1 = 0, k2 = 0;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        group[t] = g;
        if (g < a.groups) {
          k2 = key[t] > k1 ? k1 : max(k2, key[t]);
          k1 = max(k1, key[t]);
          if (--left == 0) {
            close(g, k1, k2);
            ++g, left = per / 32, k1 = k2 = 0;
          }
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < T; ++t) group[t] = (lane + 32 * t) / per;
      for (uint32_t g = 0; g < a.groups; ++g) {
        uint32_t k1 = 0, k2 = 0;
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const uint32_t k = group[t] == g ? key[t] : 0u;
          k2 = k > k1 ? k1 : max(k2, k);
          k1 = max(k1, k);
        }
        close(g, k1, k2);
      }
    }
    uint32_t kept = 0;
    for (uint32_t j = 0; j < a.top_groups; ++j) {
      const uint32_t best = __reduce_max_sync(kAll, worth);
      const uint32_t g = (uint32_t)__ffs(__ballot_sync(kAll, worth == best)) - 1;
      kept |= 1u << g;
      if (lane == g) worth = 0;
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      if (group[t] < a.groups && !((kept >> group[t]) & 1u)) key[t] = 0;
    }
  }
  // k rounds: the largest key, the lowest index among its holders.
  uint32_t id = 0;  // lane j: rank j's expert and score
  float w = 0.0f;
  for (uint32_t j = 0; j < a.k; ++j) {
    uint32_t best = 0, at = 0;
#pragma unroll
    for (int t = 0; t < T; ++t)
      if (key[t] > best) best = key[t], at = t;
    const uint32_t top = __reduce_max_sync(kAll, best);
    const uint32_t pick = __reduce_min_sync(kAll, best == top ? lane + 32 * at : kAll);
    float mine = 0.0f;
#pragma unroll
    for (int t = 0; t < T; ++t)
      if (lane + 32 * t == pick) mine = s[t], key[t] = 0;
    mine = __shfl_sync(kAll, mine, pick & 31);
    if (lane == j) id = pick, w = mine;
  }
  if (a.renorm) {
    float sum = 0.0f;
    for (uint32_t j = 0; j < a.k; ++j) {
      const float v = __shfl_sync(kAll, w, j);
      sum = j == 0 ? v : __fadd_rn(sum, v);
    }
    w = sum == 0.0f ? 0.0f : __fdiv_rn(w, sum);
  }
  if (lane < a.k) {
    a.ids[(size_t)r * a.k + lane] = id;
    a.ws[(size_t)r * a.k + lane] = __fmul_rn(w, a.factor);
  }
}

template <class E>
cudaError_t launch(const FkRouteGrouped& a, bool pdl, cudaStream_t s) {
  const dim3 grid((a.m + 3) / 4), block(128);
  if (a.n <= 64) return fk_launch_ex(route_grouped_kernel<E, 2>, grid, block, 0, s, pdl, a);
  if (a.n <= 128) return fk_launch_ex(route_grouped_kernel<E, 4>, grid, block, 0, s, pdl, a);
  if (a.n <= 256) return fk_launch_ex(route_grouped_kernel<E, 8>, grid, block, 0, s, pdl, a);
  if (a.n <= 512) return fk_launch_ex(route_grouped_kernel<E, 16>, grid, block, 0, s, pdl, a);
  return fk_launch_ex(route_grouped_kernel<E, 32>, grid, block, 0, s, pdl, a);
}

}  // namespace route
}  // namespace fk

cudaError_t fk_launch_route_grouped(const FkRouteGrouped& a, FkElem e, bool pdl, cudaStream_t s) {
  if (a.m == 0) return cudaSuccess;
  if (a.n == 0 || a.n > 1024 || a.groups == 0 || a.groups > 32 || a.n % a.groups != 0 || a.top_groups == 0 ||
      a.top_groups > a.groups || a.k == 0 || a.k > 8 || a.k > a.top_groups * (a.n / a.groups) || a.ldx < a.n)
    return cudaErrorInvalidValue;
#define FK_CALL(E) fk::route::launch<E>(a, pdl, s)
  return FK_BY_ELEM(e, FK_CALL);
#undef FK_CALL
}
