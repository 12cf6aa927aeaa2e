// Operators of a tree decoding step (gfx950): attention of a tree of drafted
// tokens over the pages, and the verification of the drafts against the
// target's probabilities.  (The append of the accepted path is
// launch_append_path in kernels.hpp.)
//
// A tree has up to 64 nodes per sequence, one per lane of a wavefront: the
// nodes a node sees are one 64-bit word, and the children of a node one
// ballot.  Node 0 is the root (the last generated token, whose K/V row is not
// in the pages yet); parents[t] < t is node t's parent, -1 that of a root.
//
// Shapes are validated by the callers (paged_cache.cpp / c_api.cpp) before
// anything is launched.
#pragma once

#include "kernels.hpp"

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace helix::hip {

constexpr std::size_t kMaxTreeNodes = 64;

//   query, out [batch, q_heads, nodes, 128]; tree_key / tree_value [batch,
//   kv_heads, nodes, 128]; parents [batch, nodes], nullptr: a chain;
//   node_counts [batch] (nodes behind a sequence's count have no row: theirs
//   in `out` stays as it was), nullptr: all; tables, lengths, pools as in
//   DecodeArgs.
struct TreeAttentionArgs {
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
  void* workspace;  // tree_workspace_bytes(...)
  std::size_t batch, q_heads, kv_heads, nodes, max_blocks, physical_blocks;
  PageFormat page_type;
};
std::size_t tree_workspace_bytes(std::size_t batch, std::size_t q_heads, std::size_t kv_heads,
                                 std::size_t nodes);
// Whether the launch's blocks of keys can be counted; where not, it fails.
bool tree_fits(const TreeAttentionArgs& a);
hipError_t launch_tree_attention(const TreeAttentionArgs& a, hipStream_t stream);

// Row strides in elements; draft == nullptr: every drafted token was certain
// to be drafted (probability 1 on it).
struct VerifyArgs {
  const float* target;  // [batch, nodes, vocab]
  std::size_t target_batch_stride, target_node_stride;
  const float* draft;   // row n: the distribution the children of node n were drawn from
  std::size_t draft_batch_stride, draft_node_stride;
  const std::int32_t* tokens;       // [batch, nodes]
  const std::int32_t* parents;      // [batch, nodes], nullptr: a chain
  const std::int32_t* node_counts;  // [batch], nullptr: all
  const float* uniforms;            // [batch, nodes]
  const float* bonus_uniforms;      // [batch]
  std::int32_t* path;               // [batch, nodes]
  std::int32_t* accepted;           // [batch]
  std::int32_t* next_token;         // [batch]
  void* workspace;                  // verify_workspace_bytes(...)
  std::size_t batch, nodes, vocab;
};
std::size_t verify_workspace_bytes(std::size_t batch, std::size_t nodes, std::size_t vocab);
hipError_t launch_verify(const VerifyArgs& a, hipStream_t stream);

}  // namespace helix::hip
