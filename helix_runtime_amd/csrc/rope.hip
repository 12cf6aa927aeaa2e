// Rotary positions.  A head's rotated part is `pairs` pairs of elements; pair i
// of the row at position p turns by the angle p f_i:
//
//   y = (a c - b s, a s + b c),  c = amplitude cos(p f_i), s = amplitude sin(p f_i),
//
// every product and sum rounded to fp32 on its own, as rope_kernel rounds them.
// The tables' angles are 64-bit numbers: at position 2^17 an fp32 angle is off by
// up to 2^-8.
#include "bf16.hpp"
#include "fp8.hpp"
#include "rope.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

namespace helix::hip {
namespace {

constexpr unsigned kThreads = 256;

// ---------------------------------------------------------------- tables ----
// A thread fills kTableRows rows of one pair: the cosine and sine of the first
// row's angle and of the step's, then a complex product a row (its error, in 64
// bits, stays far below an fp32 rounding's).  It takes two sine calls a 16 rows
// instead of one a row, which leaves the writes as the bound: 131072 rows of 64 pairs
// in 12.7 us, 5.3 TB/s, where a call a row takes 44.
constexpr int kTableRows = 16;

struct RopeTable {
  float* cosine;
  float* sine;
  long long rows, first;
  int pairs, scaling;
  double log_base, factor, original, low, high, amplitude;
  double ramp_from, ramp_width;
};

__device__ __forceinline__ double table_frequency(const RopeTable& a, int i) {
  const double share = static_cast<double>(i) / a.pairs;
  double f = exp(-share * a.log_base);
  switch (static_cast<RopeScaling>(a.scaling)) {
    case RopeScaling::kLinear: f /= a.factor; break;
    case RopeScaling::kRamp: {
      const double part = fmin(fmax((i - a.ramp_from) / a.ramp_width, 0.0), 1.0);
      f = f / a.factor * part + f * (1.0 - part);
      break;
    }
    case RopeScaling::kBands: {
      const double turns = a.original * f / 6.283185307179586;
      const double part = fmin(fmax((turns - a.low) / (a.high - a.low), 0.0), 1.0);
      f = f / a.factor * (1.0 - part) + f * part;
      break;
    }
    default: break;  // (kNtk: another base)
  }
  return f;
}

__global__ __launch_bounds__(kThreads) void rope_table_kernel(RopeTable a) {
  const long long e = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  const long long chunk = e / a.pairs;
  const int i = static_cast<int>(e - chunk * a.pairs);
  const long long row0 = chunk * kTableRows;
  if (row0 >= a.rows) return;
  const double f = table_frequency(a, i);
  double s, c, ds, dc;
  sincos(static_cast<double>(a.first + row0) * f, &s, &c);
  sincos(f, &ds, &dc);
  s *= a.amplitude;
  c *= a.amplitude;
  const int rows = static_cast<int>(min(static_cast<long long>(kTableRows), a.rows - row0));
  for (int r = 0; r < rows; ++r) {
    const long long at = (row0 + r) * a.pairs + i;
    a.cosine[at] = static_cast<float>(c);
    a.sine[at] = static_cast<float>(s);
    const double next = c * dc - s * ds;
    s = s * dc + c * ds;
    c = next;
  }
}

// ------------------------------------------------------------------ rows ----
// A division by a launch constant: n / d = (n * factor) >> 64 for n below 2^32,
// d below 2^31, factor = floor(2^64 / d) + 1.
struct Quotient {
  unsigned long long factor;
  __device__ __forceinline__ unsigned operator()(unsigned n) const {
    return static_cast<unsigned>(__umul64hi(factor, n));
  }
};
Quotient quotient(std::size_t d) {
  // (d = 1: 2^64 does not fit; the kernel never divides by 1 that way.)
  return Quotient{d == 1 ? 0 : ~0ull / d + 1};
}

struct StreamArgs {
  const float* in;
  float* out;
  void* pool;
  long long in_b, in_h, in_t, out_b, out_h, out_t;
  unsigned first_block;       // the tensor's first workgroup
  unsigned turned, per_head;  // units of a head that turn, and all of them
  unsigned per_token;
  unsigned total;
  Quotient by_head, by_token;  // by per_head and per_token
  unsigned rotary;            // elements
  unsigned pool_row, pool_from, heads;
  float scale;
};

struct RopeRowsKernelArgs {
  StreamArgs streams[3];
  int count;
  unsigned tokens;
  Quotient by_tokens;
  const std::int32_t* positions;
  const std::int32_t* starts;
  const std::int32_t* token_counts;
  const std::int64_t* slots;
  const float* cosine;
  const float* sine;
  long long table_rows, slot_limit;
  unsigned pairs, block_tokens;
  int halves, inverse;
};

template <int W>
struct Vec;
template <>
struct Vec<1> {
  using Type = float;
};
template <>
struct Vec<4> {
  using Type = float __attribute__((ext_vector_type(4)));
};

// W consecutive fp32 values as page elements at `to` (W element sizes aligned).
template <typename S, int W>
__device__ __forceinline__ void put_page(S* to, typename Vec<W>::Type v, float scale) {
  if constexpr (std::is_same_v<S, float>) {
    *reinterpret_cast<typename Vec<W>::Type*>(to) = v;
  } else if constexpr (std::is_same_v<S, unsigned short>) {
    if constexpr (W == 4) {
      *reinterpret_cast<uint2*>(to) = make_uint2(bf16_pack(v[0], v[1]), bf16_pack(v[2], v[3]));
    } else {
      *to = bf16_round(v);
    }
  } else {
    if constexpr (W == 4) {
      *reinterpret_cast<unsigned*>(to) = fp8_pack4_scaled(make_float4(v[0], v[1], v[2], v[3]), scale);
    } else {
      *to = static_cast<unsigned char>(fp8_code(v / scale));
    }
  }
}

// A thread moves one unit, 2 W elements of one row: W pairs where the row turns,
// else 2 W elements side by side.  Units of a token's heads lie one behind another,
// so a wavefront reads and writes whole cache lines and the token's table row once.
// Bound by memory: 8191 x 40 heads of 96 elements in 52 us, 4.9 TB/s; a chunk of 16 x
// 512 tokens, 32 + 8 + 8 heads of 128, rotated and appended in 92 us, 5.2 TB/s (a large
// copy: 4.7).  Element by element (W = 1, where the rows or their strides do not lie on
// 16 bytes) they take half as long again: 69 us for 45 with warm rows, 125 for 93.
template <typename S, int W>
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(RopeRowsKernelArgs a) {
#pragma clang fp contract(off)
  using V = typename Vec<W>::Type;
  // Each tensor has workgroups of its own.
  int of = 0;
  if (a.count > 1 && blockIdx.x >= a.streams[1].first_block) of = 1;
  if (a.count > 2 && blockIdx.x >= a.streams[2].first_block) of = 2;
  const StreamArgs& s = a.streams[of];
  const unsigned e = (blockIdx.x - s.first_block) * kThreads + threadIdx.x;
  if (e >= s.total) return;
  const unsigned bt = s.per_token == 1 ? e : s.by_token(e);
  const unsigned in_token = e - bt * s.per_token;
  const unsigned b = a.tokens == 1 ? bt : a.by_tokens(bt);
  const unsigned t = bt - b * a.tokens;
  if (a.token_counts != nullptr && static_cast<long long>(t) >= a.token_counts[b]) return;
  const unsigned h = s.per_head == 1 ? in_token : s.by_head(in_token);
  const unsigned u = in_token - h * s.per_head;
  const bool turns = u < s.turned;
  unsigned at0, at1;  // elements of the row
  if (turns) {
    at0 = a.halves != 0 ? u * W : u * 2 * W;
    at1 = a.halves != 0 ? s.rotary / 2 + u * W : at0 + W;
  } else {
    at0 = s.rotary + (u - s.turned) * 2 * W;
    at1 = at0 + W;
  }
  const float* const in = s.in + static_cast<long long>(b) * s.in_b +
                          static_cast<long long>(h) * s.in_h + static_cast<long long>(t) * s.in_t;
  V x = *reinterpret_cast<const V*>(in + at0);
  V y = *reinterpret_cast<const V*>(in + at1);
  if (turns) {
    long long pos = t;
    if (a.positions != nullptr) {
      pos = a.positions[bt];
    } else if (a.starts != nullptr) {
      pos += a.starts[b];
    }
    V c, sn;
    if (pos >= 0 && pos < a.table_rows) {
      const std::size_t row = static_cast<std::size_t>(pos) * a.pairs + u * W;
      c = *reinterpret_cast<const V*>(a.cosine + row);
      sn = *reinterpret_cast<const V*>(a.sine + row);
    } else {
      c = sn = V(NAN);
    }
    if (a.inverse != 0) sn = -sn;
    if constexpr (W == 1) {
      const V x0 = x;
      x = x0 * c - y * sn;
      y = x0 * sn + y * c;
    } else if (a.halves != 0) {
      const V x0 = x;
      x = x0 * c - y * sn;
      y = x0 * sn + y * c;
    } else {
      const V even = __builtin_shufflevector(x, y, 0, 2, 4, 6);
      const V odd = __builtin_shufflevector(x, y, 1, 3, 5, 7);
      const V p = even * c - odd * sn, q = even * sn + odd * c;
      x = __builtin_shufflevector(p, q, 0, 4, 1, 5);
      y = __builtin_shufflevector(p, q, 2, 6, 3, 7);
    }
  }
  if (s.out != nullptr) {
    float* const out = s.out + static_cast<long long>(b) * s.out_b +
                       static_cast<long long>(h) * s.out_h + static_cast<long long>(t) * s.out_t;
    *reinterpret_cast<V*>(out + at0) = x;
    *reinterpret_cast<V*>(out + at1) = y;
  }
  if (s.pool != nullptr) {
    const long long slot = a.slots[bt];
    if (slot < 0 || slot >= a.slot_limit) return;
    const long long block = slot / a.block_tokens;
    const unsigned row = static_cast<unsigned>(slot - block * a.block_tokens);
    S* const to = static_cast<S*>(s.pool) +
                  ((static_cast<std::size_t>(block) * s.heads + h) * a.block_tokens + row) * s.pool_row +
                  s.pool_from;
    put_page<S, W>(to + at0, x, s.scale);
    put_page<S, W>(to + at1, y, s.scale);
  }
}

// ----------------------------------------------------------------- host ----
bool aligned(const void* p, std::size_t to) {
  return reinterpret_cast<std::uintptr_t>(p) % to == 0;
}

// Whether four elements can be moved at a time everywhere.
bool vectors_fit(const RopeRowsArgs& a) {
  const std::size_t element = page_element_bytes(a.page_type);
  if (!aligned(a.cosine, 16) || !aligned(a.sine, 16) || a.pairs % 4 != 0) return false;
  for (int i = 0; i < a.count; ++i) {
    const RopeStream& s = a.streams[i];
    auto rows = [](const void* p, const Rows& r) {
      return aligned(p, 16) && r.batch % 4 == 0 && r.head % 4 == 0 && r.token % 4 == 0;
    };
    if (s.dim % 8 != 0 || s.rotary % 8 != 0 || !rows(s.in, s.in_at)) return false;
    if (s.out != nullptr && !rows(s.out, s.out_at)) return false;
    if (s.pool != nullptr &&
        (!aligned(s.pool, 4 * element) || s.pool_row % 4 != 0 || s.pool_from % 4 != 0)) {
      return false;
    }
  }
  return true;
}

template <typename S>
void launch_rows(const RopeRowsKernelArgs& k, unsigned grid, bool vectors, hipStream_t stream) {
  if (vectors) {
    rope_rows_kernel<S, 4><<<grid, kThreads, 0, stream>>>(k);
  } else {
    rope_rows_kernel<S, 1><<<grid, kThreads, 0, stream>>>(k);
  }
}

std::size_t row_elements(const RopeRowsArgs& a) {
  std::size_t n = 0;
  for (int i = 0; i < a.count; ++i) n += a.streams[i].heads * a.streams[i].dim;
  return n;
}

}  // namespace

hipError_t launch_rope_tables(const RopeTableArgs& a, hipStream_t stream) {
  const std::size_t pairs = a.rotary_dim / 2;
  if (a.rows == 0 || pairs == 0) return hipSuccess;
  RopeTable k{};
  k.cosine = a.cosine;
  k.sine = a.sine;
  k.rows = static_cast<long long>(a.rows);
  k.first = static_cast<long long>(a.first_position);
  k.pairs = static_cast<int>(pairs);
  k.scaling = static_cast<int>(a.scaling);
  const double d = static_cast<double>(a.rotary_dim);
  k.log_base = std::log(a.base);
  if (a.scaling == RopeScaling::kNtk) k.log_base += d / (d - 2.0) * std::log(a.factor);
  k.factor = a.factor;
  k.original = a.original_length;
  k.low = a.low;
  k.high = a.high;
  k.amplitude = a.amplitude;
  if (a.scaling == RopeScaling::kRamp) {
    // The pair whose wave turns `turns` times over the original length.
    auto pair_of = [&](double turns) {
      return d * std::log(a.original_length / (turns * 2.0 * 3.141592653589793)) /
             (2.0 * std::log(a.base));
    };
    k.ramp_from = std::max(std::floor(pair_of(a.high)), 0.0);
    const double to = std::min(std::ceil(pair_of(a.low)), d - 1.0);
    k.ramp_width = std::max(to - k.ramp_from, 0.001);
  }
  const std::size_t work = (a.rows + kTableRows - 1) / kTableRows * pairs;
  const std::size_t grid = (work + kThreads - 1) / kThreads;
  if (grid > 0x7fffffffu) return hipErrorInvalidValue;
  rope_table_kernel<<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(k);
  return hipGetLastError();
}

bool rope_rows_fit(const RopeRowsArgs& a) {
  // Units, of two elements at least, are counted in 32 bits.
  const std::size_t n = row_elements(a);
  return n == 0 || a.tokens == 0 ||
         (a.batch <= 0xffffffffu / a.tokens && a.batch * a.tokens <= 0xffffff00u / ((n + 1) / 2));
}

hipError_t launch_rope_rows(const RopeRowsArgs& a, hipStream_t stream) {
  if (a.batch == 0 || a.tokens == 0 || row_elements(a) == 0) return hipSuccess;
  if (!rope_rows_fit(a)) return hipErrorInvalidValue;
  const bool vectors = vectors_fit(a);
  const unsigned width = vectors ? 4 : 1;
  RopeRowsKernelArgs k{};
  k.count = a.count;
  unsigned grid = 0;
  for (int i = 0; i < a.count; ++i) {
    const RopeStream& s = a.streams[i];
    StreamArgs& o = k.streams[i];
    o.in = s.in;
    o.out = s.out;
    o.pool = s.pool;
    o.in_b = static_cast<long long>(s.in_at.batch);
    o.in_h = static_cast<long long>(s.in_at.head);
    o.in_t = static_cast<long long>(s.in_at.token);
    o.out_b = static_cast<long long>(s.out_at.batch);
    o.out_h = static_cast<long long>(s.out_at.head);
    o.out_t = static_cast<long long>(s.out_at.token);
    o.first_block = grid;
    o.turned = static_cast<unsigned>(s.rotary / (2 * width));
    o.per_head = static_cast<unsigned>(s.dim / (2 * width));
    o.by_head = quotient(std::max(o.per_head, 1u));
    o.rotary = static_cast<unsigned>(s.rotary);
    o.pool_row = static_cast<unsigned>(s.pool_row);
    o.pool_from = static_cast<unsigned>(s.pool_from);
    o.heads = static_cast<unsigned>(s.heads);
    o.scale = s.scale;
    o.per_token = static_cast<unsigned>(s.heads) * o.per_head;
    o.by_token = quotient(std::max(o.per_token, 1u));
    o.total = static_cast<unsigned>(a.batch * a.tokens) * o.per_token;
    grid += (o.total + kThreads - 1) / kThreads;
  }
  k.tokens = static_cast<unsigned>(a.tokens);
  k.by_tokens = quotient(a.tokens);
  k.positions = a.positions;
  k.starts = a.starts;
  k.token_counts = a.token_counts;
  k.slots = a.slots;
  k.cosine = a.cosine;
  k.sine = a.sine;
  k.table_rows = static_cast<long long>(a.table_rows);
  k.slot_limit = static_cast<long long>(a.physical_blocks * a.block_tokens);
  k.pairs = static_cast<unsigned>(a.pairs);
  k.block_tokens = static_cast<unsigned>(a.block_tokens);
  k.halves = a.layout == RopeLayout::kHalves ? 1 : 0;
  k.inverse = a.inverse ? 1 : 0;
  switch (a.page_type) {
    case PageType::kBF16: launch_rows<unsigned short>(k, grid, vectors, stream); break;
    case PageType::kFP8: launch_rows<unsigned char>(k, grid, vectors, stream); break;
    default: launch_rows<float>(k, grid, vectors, stream); break;
  }
  return hipGetLastError();
}

}  // namespace helix::hip
