// What both forms of attention over a latent cache share on the device: the arithmetic of
// the flat lists of tiles, matrix instructions of 16-bit terms, and a row's end.
#pragma once

#include "prefill_bmma.hpp"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstddef>

namespace helix::hip::latent_detail {

using prefill_detail::v4f;
using prefill_detail::v8bf;
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

inline std::size_t align256(std::size_t n) { return (n + 255) & ~std::size_t{255}; }

__device__ __forceinline__ long long divide(long long n, long long d) {
  // (A 64-bit division takes ten times a 32-bit one.)
  if ((n | d) >> 31 == 0) return static_cast<unsigned>(n) / static_cast<unsigned>(d);
  return n / d;
}

__device__ __forceinline__ long long uniform_long(long long v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v));
  const unsigned hi =
      __builtin_amdgcn_readfirstlane(static_cast<unsigned>(static_cast<unsigned long long>(v) >> 32));
  return static_cast<long long>(static_cast<unsigned long long>(hi) << 32 | lo);
}

// Inclusive sums over the wavefront.
__device__ __forceinline__ long long lane_scan(long long v, int lane) {
  long long sum = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long t = __shfl_up(sum, o, 64);
    if (lane >= o) sum += t;
  }
  return sum;
}

// New tokens of sequence b.
template <typename Args>
__device__ __forceinline__ int clamped_count(const Args& a, int b) {
  return a.token_counts != nullptr ? min(max(a.token_counts[b], 0), a.tokens) : a.tokens;
}

template <bool F16>
__device__ __forceinline__ v4f matrix_step(v4u a, v4u b, v4f c) {
  if constexpr (F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                  __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a),
                                                   __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
}

// What a row's outputs are multiplied by at its end: `f` over its sum.  A row that sees
// nothing has neither sum nor outputs, and is 0.  One all of whose scores are minus
// infinity has no sum either, but weights of 0 / 0: NaN.  Among partials the latter's
// reference is kNoWeights, the lowest finite number, instead of minus infinity: it weighs
// as little.
constexpr float kNoWeights = -3.402823466e38f;
__device__ __forceinline__ float row_factor(float sum, bool some, float f) {
  return sum != 0.f ? f / sum : some ? NAN : 0.f;
}
// What a partial adds to the sum of a row whose largest reference is `top`: its own sum
// times its weight, or, where all that the row sees has no weights, NaN.  (A join that
// knows `top` before it adds needs it no longer then: it takes a register less.)
__device__ __forceinline__ float part_sum(float reference, float sum, float weight, float top) {
  return sum == 0.f && reference == top && top != -INFINITY ? NAN : sum * weight;
}

}  // namespace helix::hip::latent_detail
