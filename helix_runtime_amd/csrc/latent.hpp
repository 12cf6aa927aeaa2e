// Attention over a latent cache (gfx950): pages hold one row a token, a latent
// part and a rotated part, that all query heads share.
//
// Absorbed form: a head's key is the whole row and its value the row's latent
// part, the projections around them being folded into the queries and into what
// follows.  Expanded form: each head has keys and values of its own, the rotated
// part of the keys still shared; about a third of the arithmetic a (query, key)
// pair, where the expansion is worth it: prompts.
//
// Shapes are validated by the callers (c_api.cpp) before anything is launched.
#pragma once

#include "kernels.hpp"
#include "rope.hpp"

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace helix::hip {

constexpr std::size_t kLatentRope = 64;   // rotated elements of a row
constexpr std::size_t kLatentPage = 16;   // tokens of a page
constexpr std::size_t kLatentNope = 128;  // key elements of a head without them, and of its value
constexpr bool latent_dim_supported(std::size_t n) { return n == 256 || n == 512; }

//   query [batch, q_heads, tokens, latent + 64] by query_at; out [.., latent] by
//   out_at; pool [physical_blocks, 16, latent + 64]; lengths[b] tokens of
//   sequence b lie in the pages, its token_counts[b] new ones the last: row t
//   sees the first lengths[b] - token_counts[b] + t + 1.
struct LatentArgs {
  const float* query;
  const void* pool;
  const std::uint32_t* tables;
  const std::int32_t* lengths;
  const std::int32_t* token_counts;  // null: all tokens
  float* out;
  Rows query_at, out_at;
  void* workspace;  // latent_workspace_bytes(...)
  std::size_t batch, q_heads, tokens, latent, max_blocks, physical_blocks;
  float scale;  // of the scores
  PageType page_type;
  float page_scale;
};
// Workgroups of each of the `row_blocks` units of a sequence, or 0: none of its own, all
// of them for one list.  A multiple of the XCDs keeps those that read the same pages at
// one time on one XCD (one sequence of 32768 tokens, bf16, three row blocks of 64: 52 us
// so, 54 with shares of 85, 57 with one list), unless more than three sixteenths of them
// would have nothing to do.  17 row blocks of 16 sequences of 2048 tokens, bf16, take 285 us
// on 136 workgroups and 188 on 255; 11 row blocks of 16 rows over 65536 tokens, fp8, 82 on
// 176 and 68 on 253 (with one list 195 and 80).  Between 208 and 231 workgroups it goes
// either way: 13 row blocks of 33 sequences, bf16, 247 us and 225, but as many sequences of
// one length as a multiple of eight has workgroups are best left a workgroup each (7 row
// blocks of 64 rows, 8 sequences, fp8, on 224 of them 47 us, on 252 59).
constexpr std::size_t latent_share(std::size_t groups, std::size_t row_blocks) {
  if (row_blocks <= 1 || groups / row_blocks < kXcds) return 0;
  const std::size_t share = groups / row_blocks, whole = share / kXcds * kXcds;
  return 16 * whole * row_blocks >= 13 * groups ? whole : share;
}

std::size_t latent_workspace_bytes(std::size_t batch, std::size_t q_heads, std::size_t tokens,
                                   std::size_t latent);
// Whether the launch's blocks of keys can be counted; where not, it fails.
bool latent_fits(const LatentArgs& a);
hipError_t launch_latent_attention(const LatentArgs& a, hipStream_t stream);

//   query [batch, heads, tokens, 128 + 64], key, value [batch, heads, keys, 128],
//   rope_key [batch, keys, 64] (its head stride unused), out [batch, heads,
//   tokens, 128]; key_lengths[b] (null: keys) keys of sequence b, its
//   token_counts[b] new tokens' the last.
struct ExpandedArgs {
  const float* query;
  const float* key;
  const float* rope_key;
  const float* value;
  const std::int32_t* key_lengths;
  const std::int32_t* token_counts;
  float* out;
  Rows query_at, key_at, rope_at, value_at, out_at;
  void* workspace;  // expanded_workspace_bytes(...)
  std::size_t batch, heads, tokens, keys;
  float scale;
};
std::size_t expanded_workspace_bytes(std::size_t batch, std::size_t heads, std::size_t tokens,
                                     std::size_t keys);
// Whether the launch's tiles of keys can be counted, and keys' rows are below 2^25
// numbers apart; where not, it fails.
bool expanded_fits(const ExpandedArgs& a);
hipError_t launch_expanded_attention(const ExpandedArgs& a, hipStream_t stream);

}  // namespace helix::hip
