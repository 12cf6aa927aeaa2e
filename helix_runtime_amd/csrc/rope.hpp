// Rotary positions (gfx950): tables of a context length, rows as a projection
// leaves them, and a step's new rows on their way into the pages.
//
// Shapes are validated by the callers (paged_cache.cpp / c_api.cpp) before
// anything is launched.
#pragma once

#include "kernels.hpp"

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace helix::hip {

// Which elements of a head's rotated part turn together: (2 i, 2 i + 1), or
// (i, i + half of the part).
enum class RopeLayout : int { kPairs = 0, kHalves = 1 };

// How a table's frequencies differ from base^(-2 i / rotary_dim).
enum class RopeScaling : int { kNone = 0, kLinear = 1, kNtk = 2, kRamp = 3, kBands = 4 };

struct RopeTableArgs {
  float* cosine;  // [rows, rotary_dim / 2]
  float* sine;
  std::size_t rows, first_position, rotary_dim;
  double base;
  RopeScaling scaling;
  double factor, original_length, low, high, amplitude;
};
hipError_t launch_rope_tables(const RopeTableArgs& a, hipStream_t stream);

// fp32 rows [batch, heads, tokens, dim], contiguous in their last dimension;
// strides in elements.
struct Rows {
  std::size_t batch = 0, head = 0, token = 0;
};

// One of a step's tensors: its rows, where they go as rows (out) and where as
// page elements (pool), either of which may be null.
struct RopeStream {
  const float* in = nullptr;
  float* out = nullptr;
  void* pool = nullptr;
  Rows in_at, out_at;
  std::size_t heads = 0, dim = 0;
  std::size_t rotary = 0;     // the first `rotary` elements of a row turn (0: none)
  std::size_t pool_row = 0;   // elements of a page's row of one head,
  std::size_t pool_from = 0;  // and where in it this row begins
  float scale = 1.0f;         // fp8 pages
};

// Row (b, t), t < token_counts[b], turns by table row positions[b * tokens + t],
// or (positions null) starts[b] + t, or (both null) t; outside the table the
// turned part is NaN.  Pool rows go to slots[b * tokens + t] (outside the pool:
// nowhere) of [physical_blocks, heads, block_tokens, pool_row] pages.
struct RopeRowsArgs {
  RopeStream streams[3];
  int count = 0;
  std::size_t batch = 0, tokens = 0;
  const std::int32_t* positions = nullptr;
  const std::int32_t* starts = nullptr;
  const std::int32_t* token_counts = nullptr;  // null: all tokens
  const std::int64_t* slots = nullptr;
  std::size_t physical_blocks = 0, block_tokens = 1;
  const float* cosine = nullptr;  // [table_rows, pairs]
  const float* sine = nullptr;
  std::size_t table_rows = 0, pairs = 0;
  RopeLayout layout = RopeLayout::kPairs;
  bool inverse = false;
  PageType page_type = PageType::kF32;
};
// Whether the launch's elements can be counted; where not, it fails.
bool rope_rows_fit(const RopeRowsArgs& a);
hipError_t launch_rope_rows(const RopeRowsArgs& a, hipStream_t stream);

}  // namespace helix::hip
