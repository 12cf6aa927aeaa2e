// What the kernels of a tree step's attention share, and its plain form: one
// query row by one wavefront in fp32 arithmetic, every score a sum of products
// of fp32 values, every key the row does not see left out rather than weighted
// with 0, so that infinities and NaN reach exactly the rows that see them.
// A lane holds dims 2 lane, 2 lane + 1 of the row, of a key and of its value.
#pragma once

#include "prefill_body.hpp"
#include "tree.hpp"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace helix::hip::tree_detail {

using prefill_detail::exp2_ratio;

constexpr int D = 128;
constexpr int P = 16;
constexpr float kLog2e = 1.4426950408889634f;

struct TreeKernelArgs {
  const float* query;
  const void* key_pool;
  const void* value_pool;
  const std::uint32_t* tables;
  const std::int32_t* lengths;
  const float* tree_key;
  const float* tree_value;
  const std::int32_t* parents;
  const std::int32_t* node_counts;
  float* out;
  int batch, q_heads, kv_heads, nodes, max_blocks;
  int rows;  // query rows of a (sequence, kv head): q_heads / kv_heads * nodes
  std::uint32_t physical_blocks;
  float qscale;  // log2(e) / sqrt(128)
  float k_scale, v_scale;
};

// One sequence's history, nodes and ancestor words.
struct TreeSequence {
  int hist;   // history tokens; 0 where the given length is outside the table
  int count;  // nodes
  int bad;    // length outside the table, or a page outside the pool
  // Lane t: the nodes that node t sees (itself among them), 0 for a node
  // behind the count; `broken`: node t or one of its ancestors has a parent
  // that does not come before it.
  unsigned long long seen;
  int broken;
};

__device__ __forceinline__ unsigned long long shfl64(unsigned long long v, int src) {
  const unsigned lo = __shfl(static_cast<unsigned>(v), src, 64);
  const unsigned hi = __shfl(static_cast<unsigned>(v >> 32), src, 64);
  return static_cast<unsigned long long>(hi) << 32 | lo;
}

__device__ __forceinline__ int clamped_history(const TreeKernelArgs& a, int b) {
  const int hist = a.lengths[b];
  return hist < 0 || hist > a.max_blocks * P ? -1 : hist;
}

__device__ __forceinline__ int clamped_nodes(const TreeKernelArgs& a, int b) {
  return a.node_counts != nullptr ? min(max(a.node_counts[b], 0), a.nodes) : a.nodes;
}

// Parent of node `lane` as given (-1 behind the count).
__device__ __forceinline__ int node_parent(const TreeKernelArgs& a, int b, int count, int lane) {
  if (lane >= count) return -1;
  if (a.parents == nullptr) return lane - 1;
  return a.parents[static_cast<std::size_t>(b) * a.nodes + lane];
}

// The words of all nodes from their parents, by doubling: after step k a
// lane's word holds the 2^k nearest, itself first.
__device__ __forceinline__ void tree_words(int up, int count, int lane, TreeSequence& s) {
  const bool wrong = lane < count && (up < -1 || up >= lane);
  if (wrong) up = -1;
  s.seen = lane < count ? 1ull << lane : 0ull;
#pragma unroll 1
  for (int k = 1; k < count; k *= 2) {
    const unsigned long long more = shfl64(s.seen, max(up, 0));
    const int next = __shfl(up, max(up, 0), 64);
    if (up >= 0) {
      s.seen |= more;
      up = next;
    }
  }
  s.broken = (s.seen & __ballot(wrong)) != 0;
}

__device__ __forceinline__ TreeSequence tree_sequence(const TreeKernelArgs& a, int b, int lane) {
  TreeSequence s{};
  const int hist = clamped_history(a, b);
  s.bad = hist < 0;
  s.hist = __builtin_amdgcn_readfirstlane(max(hist, 0));
  s.count = __builtin_amdgcn_readfirstlane(clamped_nodes(a, b));
  tree_words(node_parent(a, b, s.count, lane), s.count, lane, s);
  return s;
}

// Two consecutive elements at element offset e of a pool, as the values they
// stand for.
template <int PF>
__device__ __forceinline__ float2 page_pair(const void* pool, std::size_t e, float scale) {
  if constexpr (PF == 1) {
    const unsigned w = *reinterpret_cast<const unsigned*>(
        static_cast<const unsigned short*>(pool) + e);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else if constexpr (PF == 2) {
    const unsigned w =
        *reinterpret_cast<const unsigned short*>(static_cast<const unsigned char*>(pool) + e);
    const auto v = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    return make_float2(v[0] * scale, v[1] * scale);
  } else {
    return *reinterpret_cast<const float2*>(static_cast<const float*>(pool) + e);
  }
}

// Two fp32 values of a tree row as their page will hold them.
template <int PF>
__device__ __forceinline__ float2 row_pair(const float* row, float scale) {
  const float2 x = *reinterpret_cast<const float2*>(row);
  if constexpr (PF == 1) {
    return make_float2(bf16_value(bf16_round(x.x)), bf16_value(bf16_round(x.y)));
  } else if constexpr (PF == 2) {
    const float4 r = fp8_rounded(make_float4(x.x, x.y, 0.f, 0.f), scale);
    return make_float2(r.x, r.y);
  } else {
    return x;
  }
}

// Row `row` of the (sequence b, kv head) over history tokens [k0, k1) and the
// nodes [n0, n1) that its word `seen` has: its maximum (log2 units), its sum and
// this lane's two dims of its unnormalised output.  (Pages outside the pool are
// left out; the caller knows of them.)
template <int PF>
__device__ __forceinline__ void exact_row(const TreeKernelArgs& a, int b, int kvh, int row, int k0,
                                          int k1, int n0, int n1, unsigned long long seen,
                                          int lane, float2& o, float& m, float& l) {
  const std::uint32_t* const table = a.tables + static_cast<std::size_t>(b) * a.max_blocks;
  const std::size_t unit_rows =
      (static_cast<std::size_t>(b) * a.q_heads + static_cast<std::size_t>(kvh) *
                                                     (a.q_heads / a.kv_heads)) * a.nodes;
  float2 q = *reinterpret_cast<const float2*>(a.query + (unit_rows + row) * D + 2 * lane);
  q.x *= a.qscale;
  q.y *= a.qscale;
  o = make_float2(0.f, 0.f);
  m = -INFINITY;
  l = 0.f;
  auto key = [&](const float2& k, const float2& v) {
    float x = q.x * k.x + q.y * k.y;
#pragma unroll
    for (int bit = 32; bit >= 1; bit /= 2) x += __shfl_xor(x, bit, 64);
    const float mn = fmaxf(m, x);
    const float alpha = exp2_ratio(m, mn), p = exp2_ratio(x, mn);
    l = l * alpha + p;
    o.x = o.x * alpha + p * v.x;
    o.y = o.y * alpha + p * v.y;
    m = mn;
  };
  constexpr int A = 8;  // keys whose rows are loaded at once
  const float ks = PF == 2 ? a.k_scale : 1.0f, vs = PF == 2 ? a.v_scale : 1.0f;
#pragma unroll 1
  for (int j = k0; j < k1; j += A) {
    float2 k[A], v[A];
    bool ok[A];
#pragma unroll
    for (int u = 0; u < A; ++u) {
      const int pos = min(j + u, k1 - 1);
      const std::uint32_t page = table[pos / P];
      ok[u] = j + u < k1 && page < a.physical_blocks;
      k[u] = v[u] = make_float2(0.f, 0.f);
      if (ok[u]) {
        const std::size_t e =
            ((static_cast<std::size_t>(page) * a.kv_heads + kvh) * P + pos % P) * D + 2 * lane;
        k[u] = page_pair<PF>(a.key_pool, e, ks);
        v[u] = page_pair<PF>(a.value_pool, e, vs);
      }
    }
#pragma unroll
    for (int u = 0; u < A; ++u) {
      if (ok[u]) key(k[u], v[u]);
    }
  }
  const std::size_t tree0 = (static_cast<std::size_t>(b) * a.kv_heads + kvh) * a.nodes;
#pragma unroll 1
  for (int j = n0; j < n1; ++j) {
    if (((seen >> j) & 1) == 0) continue;
    key(row_pair<PF>(a.tree_key + (tree0 + j) * D + 2 * lane, ks),
        row_pair<PF>(a.tree_value + (tree0 + j) * D + 2 * lane, vs));
  }
}

}  // namespace helix::hip::tree_detail
