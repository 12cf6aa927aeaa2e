// Attention of a tree of drafted tokens over paged histories.
//
// Row t of sequence b (node t, in every query head) attends to the sequence's
// whole history and to the tree rows of its ancestors and itself:
//
//   out_t = sum_j p_tj v_j / sum_j p_tj,  p_tj = exp(q_t . k_j / sqrt(128) - m_t),
//
// j over the lengths[b] paged tokens and the nodes on t's way to its root.
// All rows of a (sequence, kv head), its query heads times the nodes, lie one
// behind another in memory.
#include "tree_exact.hpp"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace helix::hip {
namespace {

using namespace tree_detail;

// One wavefront per 16 rows of a (sequence, kv head), keys one after another.
template <int PF>
__global__ __launch_bounds__(64) void tree_rows_kernel(TreeKernelArgs a, int tiles) {
  const int lane = threadIdx.x;
  const int tile = static_cast<int>(blockIdx.x % tiles);
  const int kvh = static_cast<int>(blockIdx.x / tiles % a.kv_heads);
  const int b = static_cast<int>(blockIdx.x / tiles / a.kv_heads);
  const TreeSequence s = tree_sequence(a, b, lane);
  float2 o[16];
  float m, l;
  bool bad = s.bad;
  exact_rows<PF>(a, s, b, kvh, tile * 16, 0, s.hist, 0, s.count, lane, o, m, l, bad);
  const float inv = 1.0f / l;
  const std::size_t unit_rows =
      (static_cast<std::size_t>(b) * a.q_heads + static_cast<std::size_t>(kvh) *
                                                     (a.q_heads / a.kv_heads)) * a.nodes;
  const unsigned long long broken = __ballot(s.broken);
  const unsigned long long no_result = __ballot(m == -INFINITY);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = tile * 16 + i;
    const int node = row % a.nodes;
    if (row >= a.rows || node >= s.count) continue;
    const float sc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(inv), 4 * i));
    float2 r = make_float2(o[i].x * sc, o[i].y * sc);
    if (bad || ((no_result >> (4 * i)) & 1) != 0 || ((broken >> node) & 1) != 0) {
      r = make_float2(NAN, NAN);
    }
    *reinterpret_cast<float2*>(a.out + (unit_rows + row) * D + 2 * lane) = r;
  }
}

}  // namespace

std::size_t tree_workspace_bytes(std::size_t, std::size_t, std::size_t, std::size_t) { return 256; }

hipError_t launch_tree_attention(const TreeAttentionArgs& a, hipStream_t stream) {
  if (a.batch == 0 || a.nodes == 0) return hipSuccess;
  TreeKernelArgs k{};
  k.query = a.query;
  k.key_pool = a.key_pool;
  k.value_pool = a.value_pool;
  k.tables = a.tables;
  k.lengths = a.lengths;
  k.tree_key = a.tree_key;
  k.tree_value = a.tree_value;
  k.parents = a.parents;
  k.node_counts = a.node_counts;
  k.out = a.out;
  k.batch = static_cast<int>(a.batch);
  k.q_heads = static_cast<int>(a.q_heads);
  k.kv_heads = static_cast<int>(a.kv_heads);
  k.nodes = static_cast<int>(a.nodes);
  k.max_blocks = static_cast<int>(a.max_blocks);
  k.rows = static_cast<int>(a.q_heads / a.kv_heads * a.nodes);
  k.physical_blocks = static_cast<std::uint32_t>(a.physical_blocks);
  k.qscale = kLog2e / sqrtf(static_cast<float>(D));
  k.k_scale = a.page_type.k_scale;
  k.v_scale = a.page_type.v_scale;
  const int tiles = (k.rows + 15) / 16;
  const dim3 grid(static_cast<unsigned>(a.batch * a.kv_heads * static_cast<std::size_t>(tiles)));
  switch (a.page_type.type) {
    case PageType::kBF16: tree_rows_kernel<1><<<grid, 64, 0, stream>>>(k, tiles); break;
    case PageType::kFP8: tree_rows_kernel<2><<<grid, 64, 0, stream>>>(k, tiles); break;
    default: tree_rows_kernel<0><<<grid, 64, 0, stream>>>(k, tiles); break;
  }
  return hipGetLastError();
}

}  // namespace helix::hip
