// Expanded attention of a latent cache's prompts:
//
//   out_ht = sum_j p_j v_hj / sum_j p_j,
//   p_j = exp(scale (q_ht[:128] . k_hj + q_ht[128:] . r_j) - m),
//
// j over the keys that row t sees, r_j the rotated part of key j that every head
// shares.
//
// One wavefront a row: a lane holds elements lane and lane + 64 of a head's key
// and value and element lane of the shared part.
#include "latent.hpp"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace helix::hip {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct ExpandedKernelArgs {
  const float* query;
  const float* key;
  const float* rope_key;
  const float* value;
  const std::int32_t* key_lengths;
  const std::int32_t* token_counts;
  float* out;
  Rows query_at, key_at, rope_at, value_at, out_at;
  int batch, heads, tokens, keys;
  float qscale;  // log2(e) * scale
};

__global__ __launch_bounds__(256) void expanded_row_kernel(ExpandedKernelArgs a) {
  const int lane = threadIdx.x & 63;
  const long long rows = static_cast<long long>(a.batch) * a.heads * a.tokens;
  const long long r = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const int t = static_cast<int>(r % a.tokens);
  const int h = static_cast<int>(r / a.tokens % a.heads);
  const int b = static_cast<int>(r / a.tokens / a.heads);
  int count = a.tokens;
  if (a.token_counts != nullptr) count = min(max(a.token_counts[b], 0), a.tokens);
  if (t >= count) return;
  const int length = a.key_lengths != nullptr ? a.key_lengths[b] : a.keys;
  const bool bad = length < 0 || length > a.keys;
  const int seen = bad ? 0 : max(length - count + t + 1, 0);
  const float* const q = a.query + b * a.query_at.batch + h * a.query_at.head + t * a.query_at.token;
  const float* const key = a.key + b * a.key_at.batch + h * a.key_at.head;
  const float* const rope = a.rope_key + b * a.rope_at.batch;
  const float* const value = a.value + b * a.value_at.batch + h * a.value_at.head;
  const float q0 = q[lane] * a.qscale, q1 = q[lane + 64] * a.qscale, q2 = q[lane + 128] * a.qscale;
  float o0 = 0.f, o1 = 0.f, m = -INFINITY, l = 0.f;
  for (int j = 0; j < seen; ++j) {
    const float* const k = key + j * a.key_at.token;
    const float* const v = value + j * a.value_at.token;
    float x = q0 * k[lane] + q1 * k[lane + 64] + q2 * rope[j * a.rope_at.token + lane];
#pragma unroll
    for (int bit = 32; bit >= 1; bit /= 2) x += __shfl_xor(x, bit, 64);
    const float mn = fmaxf(m, x);
    const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    const float p = x == mn ? 1.0f : __builtin_amdgcn_exp2f(x - mn);
    l = l * alpha + p;
    o0 = o0 * alpha + p * v[lane];
    o1 = o1 * alpha + p * v[lane + 64];
    m = mn;
  }
  const float f = bad ? NAN : seen == 0 ? 0.f : 1.0f / l;
  float* const out = a.out + b * a.out_at.batch + h * a.out_at.head + t * a.out_at.token;
  out[lane] = o0 * f;
  out[lane + 64] = o1 * f;
}

}  // namespace

std::size_t expanded_workspace_bytes(std::size_t, std::size_t, std::size_t, std::size_t) {
  return 16;
}

hipError_t launch_expanded_attention(const ExpandedArgs& a, hipStream_t stream) {
  if (a.batch == 0 || a.heads == 0 || a.tokens == 0) return hipSuccess;
  ExpandedKernelArgs k{};
  k.query = a.query;
  k.key = a.key;
  k.rope_key = a.rope_key;
  k.value = a.value;
  k.key_lengths = a.key_lengths;
  k.token_counts = a.token_counts;
  k.out = a.out;
  k.query_at = a.query_at;
  k.key_at = a.key_at;
  k.rope_at = a.rope_at;
  k.value_at = a.value_at;
  k.out_at = a.out_at;
  k.batch = static_cast<int>(a.batch);
  k.heads = static_cast<int>(a.heads);
  k.tokens = static_cast<int>(a.tokens);
  k.keys = static_cast<int>(a.keys);
  k.qscale = kLog2e * a.scale;
  const std::size_t rows = a.batch * a.heads * a.tokens;
  if (rows > (std::size_t{1} << 32)) return hipErrorInvalidValue;
  expanded_row_kernel<<<static_cast<unsigned>((rows + 3) / 4), 256, 0, stream>>>(k);
  return hipGetLastError();
}

}  // namespace helix::hip
