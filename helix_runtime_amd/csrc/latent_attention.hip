// Absorbed attention over a latent cache:
//
//   out_ht = sum_j p_j c_j[:L] / sum_j p_j,  p_j = exp(scale q_ht . c_j - m),
//
// j over the tokens that row t sees, c_j the row of L + 64 elements that every
// head shares.
//
// One wavefront a row: a lane holds every 64th element of the query, of a key and
// of the output, one pass over the keys.
#include "bf16.hpp"
#include "fp8.hpp"
#include "latent.hpp"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace helix::hip {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int P = static_cast<int>(kLatentPage);

struct LatentKernelArgs {
  const float* query;
  const void* pool;
  const std::uint32_t* tables;
  const std::int32_t* lengths;
  const std::int32_t* token_counts;
  float* out;
  Rows query_at, out_at;
  int batch, q_heads, tokens, max_blocks;
  std::uint32_t physical_blocks;
  float qscale;  // log2(e) * scale
  float page_scale;
};

template <int PF>
__device__ __forceinline__ float page_value(const void* pool, std::size_t e, float scale) {
  if constexpr (PF == 1) {
    return bf16_value(static_cast<const unsigned short*>(pool)[e]);
  } else if constexpr (PF == 2) {
    return fp8_value(static_cast<const unsigned char*>(pool)[e], scale);
  } else {
    return static_cast<const float*>(pool)[e];
  }
}

template <int PF, int L>
__global__ __launch_bounds__(256) void latent_row_kernel(LatentKernelArgs a) {
  constexpr int W = L + static_cast<int>(kLatentRope);
  constexpr int NK = W / 64, NV = L / 64;
  const int lane = threadIdx.x & 63;
  const long long rows = static_cast<long long>(a.batch) * a.q_heads * a.tokens;
  const long long r = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const int t = static_cast<int>(r % a.tokens);
  const int h = static_cast<int>(r / a.tokens % a.q_heads);
  const int b = static_cast<int>(r / a.tokens / a.q_heads);
  int count = a.tokens;
  if (a.token_counts != nullptr) count = min(max(a.token_counts[b], 0), a.tokens);
  if (t >= count) return;
  const int length = a.lengths[b];
  bool bad = length < 0 || length > a.max_blocks * P;
  const int seen = bad ? 0 : max(length - count + t + 1, 0);
  const float* const q = a.query + b * a.query_at.batch + h * a.query_at.head + t * a.query_at.token;
  float qv[NK], o[NV];
#pragma unroll
  for (int i = 0; i < NK; ++i) qv[i] = q[64 * i + lane] * a.qscale;
#pragma unroll
  for (int i = 0; i < NV; ++i) o[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < seen; ++j) {
    const std::uint32_t page = a.tables[static_cast<std::size_t>(b) * a.max_blocks + j / P];
    if (page >= a.physical_blocks) {
      bad = true;
      break;
    }
    const std::size_t e = (static_cast<std::size_t>(page) * P + j % P) * W + lane;
    float k[NK], x = 0.f;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      k[i] = page_value<PF>(a.pool, e + 64 * i, a.page_scale);
      x += qv[i] * k[i];
    }
#pragma unroll
    for (int bit = 32; bit >= 1; bit /= 2) x += __shfl_xor(x, bit, 64);
    const float mn = fmaxf(m, x);
    const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    const float p = x == mn ? 1.0f : __builtin_amdgcn_exp2f(x - mn);
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i] = o[i] * alpha + p * k[i];
    m = mn;
  }
  const float f = bad ? NAN : seen == 0 ? 0.f : 1.0f / l;
  float* const out = a.out + b * a.out_at.batch + h * a.out_at.head + t * a.out_at.token;
#pragma unroll
  for (int i = 0; i < NV; ++i) out[64 * i + lane] = seen == 0 && !bad ? 0.f : o[i] * f;
}

template <int PF>
void launch_rows(const LatentKernelArgs& k, std::size_t latent, hipStream_t stream) {
  const long long rows = static_cast<long long>(k.batch) * k.q_heads * k.tokens;
  const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
  if (latent == 512) {
    latent_row_kernel<PF, 512><<<grid, 256, 0, stream>>>(k);
  } else {
    latent_row_kernel<PF, 256><<<grid, 256, 0, stream>>>(k);
  }
}

}  // namespace

std::size_t latent_workspace_bytes(std::size_t, std::size_t, std::size_t, std::size_t) { return 16; }

bool latent_fits(const LatentArgs& a) {
  return a.batch == 0 || a.q_heads == 0 || a.tokens == 0 ||
         a.batch * a.q_heads <= (std::size_t{1} << 32) / a.tokens;
}

hipError_t launch_latent_attention(const LatentArgs& a, hipStream_t stream) {
  if (a.batch == 0 || a.q_heads == 0 || a.tokens == 0) return hipSuccess;
  if (!latent_fits(a)) return hipErrorInvalidValue;
  LatentKernelArgs k{};
  k.query = a.query;
  k.pool = a.pool;
  k.tables = a.tables;
  k.lengths = a.lengths;
  k.token_counts = a.token_counts;
  k.out = a.out;
  k.query_at = a.query_at;
  k.out_at = a.out_at;
  k.batch = static_cast<int>(a.batch);
  k.q_heads = static_cast<int>(a.q_heads);
  k.tokens = static_cast<int>(a.tokens);
  k.max_blocks = static_cast<int>(a.max_blocks);
  k.physical_blocks = static_cast<std::uint32_t>(a.physical_blocks);
  k.qscale = kLog2e * a.scale;
  k.page_scale = a.page_scale;
  switch (a.page_type) {
    case PageType::kBF16: launch_rows<1>(k, a.latent, stream); break;
    case PageType::kFP8: launch_rows<2>(k, a.latent, stream); break;
    default: launch_rows<0>(k, a.latent, stream); break;
  }
  return hipGetLastError();
}

}  // namespace helix::hip
